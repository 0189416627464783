"""The int8 operators on a GPU against their definition (include/sigcomp_b200.h) in 64 bits.

The definition fixes every rounding, so results are compared for equality, without a tolerance.  Whole
sums are exact in float64 (k * 128 * 128 < 2**31), a product of two float32 is exact in float64, and the
one sum that is not (the bias) is rounded to odd in float64 first, which makes the following rounding to
float32 the only one that counts (53 >= 24 + 2 bits).
"""

import numpy as np
import pytest
import torch

from sigcomp_b200 import _lib

pytestmark = pytest.mark.gpu

SMALLEST = np.float32(2.0 ** -100)
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from sigcomp_b200 import int8
    return int8


# ---- the definition ----------------------------------------------------------------------------

def want_quantized(x):
    """(q, scales) of float32 rows."""
    x = np.asarray(x, dtype=np.float32)
    q = np.zeros(x.shape, dtype=np.int8)
    scales = np.full(x.shape[0], np.nan, dtype=np.float32)
    fine = np.isfinite(x).all(axis=1)
    top = np.maximum(np.abs(x[fine]).max(axis=1), SMALLEST)
    scales[fine] = top / np.float32(127)
    r = (np.float32(127) / top).astype(np.float64)
    q[fine] = np.rint(x[fine].astype(np.float64) * r[:, None]).astype(np.int8)
    return q, scales


def add_to_odd(p, b):
    """p + b in float64, rounded to odd."""
    s = p + b
    bb = s - p
    err = (p - (s - bb)) + (b - bb)
    even = (s.view(np.int64) & 1) == 0
    return np.where((err != 0) & even, np.nextafter(s, np.where(err > 0, np.inf, -np.inf)), s)


def want_linear(q, scales, w, ws, bias, relu):
    """Float32 results of int8 rows."""
    total = (q.astype(np.float64) @ w.astype(np.float64).T).astype(np.float32)
    t = (total * scales.astype(np.float32)[:, None]).astype(np.float64)
    p = t * ws.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        y = (p if bias is None else add_to_odd(p, np.broadcast_to(bias.astype(np.float64), p.shape))).astype(np.float32)
    return np.where(y < 0, np.float32(0), y) if relu else y


def same(got, want):
    got, want = got.cpu(), torch.from_numpy(np.ascontiguousarray(want)).to(got.dtype)
    assert got.shape == want.shape
    fine = (got == want) | (torch.isnan(got) & torch.isnan(want)) if got.dtype.is_floating_point else got == want
    bad = (~fine).nonzero()
    assert len(bad) == 0, (f"{len(bad)} of {got.numel()} differ, first at {bad[0].tolist()}: "
                           f"{got[tuple(bad[0])].item()} instead of {want[tuple(bad[0])].item()}")


# ---- inputs ------------------------------------------------------------------------------------

def float_rows(rows, cols, dtype, seed, pad=0, offset=0):
    rng = np.random.default_rng(seed)
    x = rng.normal(0, 1, size=(rows, cols + pad + offset)) * np.exp(rng.normal(0, 2, size=(rows, 1)))
    if rows > 2:
        x[rows // 2] = 0
    return torch.from_numpy(x.astype(np.float32)).to(dtype).to(DEV)[:, offset:offset + cols]


def int8_rows(rows, cols, seed, stride=None):
    rng = np.random.default_rng(seed)
    stride = stride or -(-cols // 16) * 16
    q = rng.integers(-128, 128, size=(rows, stride), dtype=np.int64).astype(np.int8)
    return torch.from_numpy(q).to(DEV)[:, :cols]


def layer(n, k, seed, bias=True, stride=None):
    rng = np.random.default_rng(seed)
    w = int8_rows(n, k, seed + 1, stride)
    ws = (rng.uniform(0.5, 1.5, n) * 2e-4 / np.sqrt(k)).astype(np.float32)
    b = rng.normal(0, 0.5, n).astype(np.float32) if bias else None
    return w, torch.from_numpy(ws).to(DEV), None if b is None else torch.from_numpy(b).to(DEV)


def scales_of(rows, seed):
    return torch.from_numpy(np.random.default_rng(seed).uniform(0.2, 3, rows).astype(np.float32)).to(DEV)


def host(t):
    return None if t is None else t.float().cpu().numpy() if t.dtype.is_floating_point else t.cpu().numpy()


# ---- quantise ----------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (33, 64), (5, 250), (9, 256), (4, 512), (3, 513), (7, 1024),
                                       (2, 2047), (3, 4096), (2, 8192), (1, 8193), (2, 20000), (1, 40001), (1000, 33)])
@pytest.mark.parametrize("pad,offset", [(0, 0), (1, 0), (8, 8), (5, 3)])
def test_quantize(ops, dtype, rows, cols, pad, offset):
    x = float_rows(rows, cols, dtype, rows * 31 + cols, pad, offset)
    q, s = ops.quantize_tokens(x)
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and q.stride(0) % 16 == 0
    wq, wscale = want_quantized(host(x))
    same(q, wq)
    same(s, wscale)
    for out in (torch.float32, torch.float16, torch.bfloat16):
        y = ops.dequantize_tokens(q, s, dtype=out)
        with np.errstate(over="ignore"):
            same(y, torch.from_numpy(wq.astype(np.float32) * wscale[:, None]).to(out).float().numpy())


def test_quantize_ties_and_extremes(ops):
    """Halves go to the even number; denormal, huge, infinite and NaN values; rows of zeros."""
    ties = np.arange(-127, 127, dtype=np.float32) + 0.5
    tiny = np.array([2.0 ** -149, -(2.0 ** -126), 2.0 ** -101], dtype=np.float32)
    rows = np.zeros((12, 256), dtype=np.float32)
    rows[0, :254], rows[0, 254] = ties, 127            # r = 1 exactly
    rows[1, :254], rows[1, 254] = ties * 4, -508
    rows[2, :3] = tiny
    rows[3, :3] = [np.finfo(np.float32).max, -1, np.finfo(np.float32).max / 254]
    rows[4, 7] = np.inf
    rows[5, 255] = -np.inf
    rows[6, 100] = np.nan
    rows[7, 31], rows[7, 3] = np.nan, np.inf
    rows[8] = -0.0
    rows[9, :] = 2.0 ** -100
    rows[10, 5] = -3e-39
    rows[11, :] = 1e30
    x = torch.from_numpy(rows).to(DEV)
    q, s = ops.quantize_tokens(x)
    wq, ws = want_quantized(rows)
    same(q, wq)
    same(s, ws)
    assert torch.isnan(s[4:8]).all() and not q[4:8].any()
    assert s[8] > 0 and not q[8].any()
    y = ops.dequantize_tokens(q, s)
    assert torch.isnan(y[4:8]).all() and not torch.isnan(y[8]).any()


def test_quantize_leaves_the_bytes_between_rows(ops):
    """Bytes behind a row's end, up to the next row's start, stay."""
    x = float_rows(5, 37, torch.float32, 3)
    q = torch.full((6, 48), 77, dtype=torch.int8, device=DEV)
    s = torch.full((6,), 5.0, device=DEV)
    rc = _lib.load().sc_quantize_tokens_device(0, x.data_ptr(), 0, 5, 37, x.stride(0), q.data_ptr(), 48, s.data_ptr(),
                                               torch.cuda.current_stream().cuda_stream)
    _lib.check(rc)
    same(q[:5, :37], want_quantized(host(x))[0])
    assert (q[:, 37:] == 77).all() and (q[5] == 77).all() and s[5] == 5


def test_batch_dimensions_and_views(ops):
    x = float_rows(24, 96, torch.bfloat16, 5)
    q, s = ops.quantize_tokens(x)
    for view in (x.view(2, 3, 4, 96), x[0], x[:0], x.view(2, 12, 96).transpose(0, 1), x.t().contiguous().t()):
        vq, vs = ops.quantize_tokens(view)
        assert vq.shape == view.shape and vs.shape == view.shape[:-1]
        wq, ws = want_quantized(host(view.reshape(-1, 96)))
        same(vq.reshape(-1, 96), wq)
        same(vs.reshape(-1), ws)
        y = ops.dequantize_tokens(vq, vs, dtype=torch.float16)
        assert y.shape == view.shape
    one = x[:1].expand(6, 96)
    same(ops.quantize_tokens(one)[0], np.repeat(host(q[:1]), 6, axis=0))
    same(ops.dequantize_tokens(q, 0.25), host(q) * np.float32(0.25))


# ---- product -----------------------------------------------------------------------------------

SIZES = [(1, 1, 1), (1, 64, 512), (1, 8192, 512), (1, 4097, 130), (2, 17, 3), (3, 512, 512), (5, 1000, 33),
         (8, 8192, 96), (9, 96, 257), (16, 512, 512), (17, 4096, 640), (31, 129, 100), (64, 8192, 512), (65, 512, 256),
         (100, 300, 1100), (127, 128, 128), (128, 128, 256), (129, 1, 257), (200, 2048, 64), (255, 511, 511),
         (257, 129, 513), (300, 1000, 777), (640, 512, 512), (1001, 96, 2304), (2049, 640, 300), (5000, 512, 256),
         (20000, 64, 16), (40000, 128, 512), (9001, 64, 1300), (20000, 300, 700), (30011, 48, 2049)]


@pytest.mark.parametrize("rows,k,n", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_linear(ops, rows, k, n, dtype):
    q, s = int8_rows(rows, k, rows + k), scales_of(rows, n)
    relu, bias = (rows + n) % 2 == 1, (rows + k) % 3 != 0
    w, ws, b = layer(n, k, n, bias)
    y = ops.int8_linear(q, w, ws, b, x_scales=s, relu=relu, dtype=dtype)
    assert y.dtype == dtype and y.stride(0) * y.element_size() % 16 == 0
    same(y, want_linear(host(q), host(s), host(w), host(ws), host(b), relu))


@pytest.mark.parametrize("rows,k,n", SIZES)
def test_linear_requant(ops, rows, k, n):
    q, s = int8_rows(rows, k, rows + k + 1), scales_of(rows, n)
    relu = (k + n) % 2 == 0
    w, ws, b = layer(n, k, n + 3, rows % 4 != 0)
    y = want_linear(host(q), host(s), host(w), host(ws), host(b), relu)
    yq, ys = ops.int8_linear_requant(q, s, w, ws, b, relu=relu)
    wq, wscale = want_quantized(y)
    same(ys, wscale)
    same(yq, wq)
    logits = ops.int8_linear_requant(q, s, w, ws, b, relu=relu, output_scale=0.011)
    assert logits.dtype == torch.int8
    same(logits, np.clip(np.rint(y / np.float32(0.011)), -128, 127).astype(np.int8))


@pytest.mark.parametrize("rows,k,n", [(1, 8192, 512), (1, 33, 7), (4, 4096, 512), (24, 4096, 256), (130, 1000, 77),
                                      (1, 20000, 20), (600, 512, 512)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("pad", [0, 3])
def test_linear_of_float_rows(ops, rows, k, n, dtype, pad):
    x = float_rows(rows, k, dtype, rows + n, pad)
    w, ws, b = layer(n, k, 5)
    y = ops.int8_linear(x, w, ws, b)
    assert y.dtype == dtype
    q, s = want_quantized(host(x))
    with np.errstate(over="ignore"):
        same(y, want_linear(q, s, host(w), host(ws), host(b), False))


@pytest.mark.parametrize("rows,k,n", [(1, 100, 50), (8, 64, 64), (70, 129, 130), (300, 513, 300)])
@pytest.mark.parametrize("xstride,wstride,shift", [(0, 0, 0), (1, 3, 0), (0, 0, 1), (16, 7, 4), (13, 16, 8)])
def test_strides_and_alignment(ops, rows, k, n, xstride, wstride, shift):
    """Rows any distance apart, starting at any byte."""
    q = int8_rows(rows, k + shift, 1, k + shift + xstride)[:, shift:]
    w, ws, b = layer(n, k + shift, 2, stride=k + shift + wstride)
    w = w[:, shift:]
    s = scales_of(rows, 3)
    want = want_linear(host(q), host(s), host(w), host(ws), host(b), False)
    same(ops.int8_linear(q, w, ws, b, x_scales=s), want)
    same(ops.int8_linear_requant(q, s, w, ws, b)[0], want_quantized(want)[0])
    # columns apart, a row repeated, a row of the weight repeated
    t = torch.zeros((k, rows), dtype=torch.int8, device=DEV)
    t.copy_(q.t())
    same(ops.int8_linear(t.t(), w, ws, b, x_scales=s), want)
    same(ops.int8_linear(q[:1].expand(5, k), w, ws, b, x_scales=s[:1].expand(5)), np.repeat(want[:1], 5, axis=0))
    same(ops.int8_linear(q, w[:1].expand(n, k), ws[:1].expand(n), b[:1].expand(n), x_scales=s),
         np.repeat(want[:, :1], n, axis=1))
    # scales and bias that start anywhere
    ws2, b2, s2 = (torch.cat([v[:1], v])[1:] for v in (ws, b, s))
    same(ops.int8_linear(q, w, ws2, b2, x_scales=s2), want)


def test_longest_sums(ops):
    """The largest whole sums: 131,071 products of 128 * 128 stay below 2**31."""
    k = 131071
    q = torch.full((3, k), -128, dtype=torch.int8, device=DEV)
    q[1] = 127
    w = torch.full((20, k), -128, dtype=torch.int8, device=DEV)
    w[3:9] = 127
    w[::2, ::7] = 3
    s, ws = torch.ones(3, device=DEV), torch.ones(20, device=DEV)
    want = want_linear(host(q), host(s), host(w), host(ws), None, False)
    assert want.max() == np.float32(k * 128 * 128)
    same(ops.int8_linear(q, w, ws, x_scales=s), want)
    same(ops.int8_linear(q.repeat(50, 1), w, ws, x_scales=s.repeat(50)), np.tile(want, (50, 1)))


@pytest.mark.parametrize("rows", [4, 40, 700])
def test_rows_that_cannot_be_quantised(ops, rows):
    """A row with an infinity or a NaN is NaN in the result, ReLU included, and no other row is."""
    x = float_rows(rows, 256, torch.bfloat16, 7)
    x[1, 5], x[3, 255] = float("inf"), float("nan")
    w, ws, b = layer(300, 256, 9)
    for relu in (False, True):
        y = ops.int8_linear(x, w, ws, b, relu=relu)
        bad = torch.isnan(y).all(dim=1)
        assert bad[1] and bad[3] and not torch.isnan(y[~bad]).any() and int(bad.sum()) == 2
    q, s = ops.quantize_tokens(x)
    yq, ys = ops.int8_linear_requant(q, s, w, ws, b, relu=True)
    assert torch.isnan(ys[[1, 3]]).all() and not yq[[1, 3]].any() and int(torch.isnan(ys).sum()) == 2
    logits = ops.int8_linear_requant(q, s, w, ws, b, output_scale=0.5)
    assert not logits[[1, 3]].any()
    # a NaN or an infinity in a channel's scale or bias
    ws2, b2 = ws.clone(), b.clone()
    ws2[7], b2[11] = float("nan"), float("inf")
    y = ops.int8_linear(q, w, ws2, b2, x_scales=s.nan_to_num(1.0))
    assert torch.isnan(y[:, 7]).all() and torch.isinf(y[:, 11]).all() and int((~torch.isfinite(y)).sum()) == 2 * rows
    ys = ops.int8_linear_requant(q, s.nan_to_num(1.0), w, ws2, b2)[1]
    assert torch.isnan(ys).all()


@pytest.mark.parametrize("k,n", [(8192, 512), (512, 512), (512, 256), (300, 700)])
def test_results_do_not_depend_on_the_batch(ops, k, n):
    """What a batch gives for a row, the row alone gives, bit for bit: an encoder works in batches, a
    decoder token by token."""
    x = float_rows(1100, k, torch.bfloat16, 1)
    w, ws, b = layer(n, k, 2)
    q, s = ops.quantize_tokens(x)
    y = ops.int8_linear(x, w, ws, b, dtype=torch.float32)
    yq, ys = ops.int8_linear_requant(q, s, w, ws, b, relu=True)
    for rows in (1, 2, 7, 16, 33, 130, 500):
        i = 1100 - rows
        assert torch.equal(ops.int8_linear(x[i:], w, ws, b, dtype=torch.float32), y[i:])
        assert torch.equal(ops.int8_linear(q[i:], w, ws, b, x_scales=s[i:]), y[i:])
        rq, rs = ops.int8_linear_requant(q[i:], s[i:], w, ws, b, relu=True)
        assert torch.equal(rq, yq[i:]) and torch.equal(rs, ys[i:])


def test_no_rows(ops):
    w, ws, b = layer(40, 64, 1)
    assert ops.int8_linear(torch.zeros((0, 64), device=DEV), w, ws, b).shape == (0, 40)
    q, s = ops.quantize_tokens(torch.zeros((2, 0, 64), device=DEV))
    assert q.shape == (2, 0, 64) and s.shape == (2, 0)
    q, s = ops.int8_linear_requant(q, s, w, ws, b)
    assert q.shape == (2, 0, 40) and s.shape == (2, 0)
    assert ops.dequantize_tokens(q, s).shape == (2, 0, 40)


# ---- streams, graphs, a run of them ------------------------------------------------------------

def _chain(ops, x, layers, scale):
    q, s = ops.quantize_tokens(x)
    for i, l in enumerate(layers[:-1]):
        q, s = ops.int8_linear_requant(q, s, *l, relu=True)
    return ops.int8_linear_requant(q, s, *layers[-1], output_scale=scale)


@pytest.mark.parametrize("rows", [1, 50, 3000])
def test_other_streams_and_graphs(ops, rows):
    """A side stream, two captured graphs replayed at the same time, an eager call between replays."""
    layers = [layer(512, 1024, 1), layer(512, 512, 2), layer(300, 512, 3)]
    xs = [float_rows(rows, 1024, torch.bfloat16, seed) for seed in (1, 2, 3)]
    want = [_chain(ops, x, layers, 0.02).clone() for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _chain(ops, xs[1], layers, 0.02)
    side.synchronize()
    assert torch.equal(got, want[1])
    graphs, ins, outs = [], [x.clone() for x in xs[:2]], []
    for x in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_chain(ops, x, layers, 0.02))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(4):
        for i, (g, st) in enumerate(zip(graphs, streams)):
            ins[i].copy_(xs[(turn + i) % 3])
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        eager = _chain(ops, xs[2], layers, 0.02)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[2])
        for i in range(2):
            assert torch.equal(outs[i], want[(turn + i) % 3])


def test_entropy_model_of_int8_layers_codes_and_decodes(ops):
    """A model with scales for each token and channel in front of the framework's range coder: windows of
    embeddings, three layers, int8 logits.  Encoded from the logits of one batch of all steps, decoded with
    logits computed window by window in batches of one row each and of all streams."""
    import ctypes
    from sigcomp_b200.codec import B200Compression
    from sigcomp_b200.model import random_model
    model = random_model(3)
    codec = B200Compression(chunk_len=2048, gpu=0, model=model)
    streams, steps, window = 6, 40, model.window_size
    rng = np.random.default_rng(0)
    table = torch.from_numpy(model.embedding.astype(np.float32)).to(torch.bfloat16).to(DEV)
    layers = [layer(512, window * model.emb_dim, 1), layer(512, 512, 2), layer(256, 512, 3)]
    symbols = rng.integers(0, 256, size=(streams, steps)).astype(np.uint8)
    padded = np.concatenate([np.full((streams, window), 256), symbols.astype(np.int64)], axis=1)
    ids = np.stack([padded[:, t:t + window] for t in range(steps)], axis=1)            # [streams, steps, window]
    x = table[torch.from_numpy(ids).to(DEV)].reshape(streams, steps, -1)
    scale = float(model.output_scale)
    logits = _chain(ops, x, layers, scale)
    assert logits.shape == (streams, steps, 256) and logits.float().std() > 1
    flat = logits.contiguous().view(-1, 256)
    off = torch.arange(0, streams * steps + 1, steps, dtype=torch.int64, device=DEV)
    sym = torch.from_numpy(symbols.reshape(-1)).to(DEV)
    words = torch.zeros(streams * (steps + 2), dtype=torch.int32, device=DEV)
    woff = torch.zeros(streams + 1, dtype=torch.int64, device=DEV)
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    _lib.check(codec._lib.sc_encode_logits_device(codec.handle, p(flat), p(sym), p(off), streams, p(words),
                                                  words.numel(), p(woff), None, st))
    # decoder's logits: one step of all streams at a time, and one row at a time
    by_step = torch.stack([_chain(ops, x[:, t], layers, scale) for t in range(steps)], dim=1).contiguous()
    assert torch.equal(by_step, logits)
    by_row = torch.stack([_chain(ops, x[2, t], layers, scale) for t in range(steps)])
    assert torch.equal(by_row, logits[2])
    back = torch.zeros(streams * steps, dtype=torch.uint8, device=DEV)
    _lib.check(codec._lib.sc_decode_logits_device(codec.handle, p(by_step.view(-1, 256)), p(off), p(words), p(woff),
                                                  streams, p(back), None, st))
    assert np.array_equal(back.cpu().numpy().reshape(streams, steps), symbols)
    codec.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(5, 3), (300, 8), (1000, 21), (700, 130), (33, 1023), (9, 4099), (4, 16383)])
@pytest.mark.parametrize("shift", [0, 1, 2, 5])
def test_rows_at_any_address(ops, dtype, rows, cols, shift):
    """Rows of x, of q and of the values that start at any element, read and written whole: nothing before the
    first row, between rows or behind the last one is touched."""
    x = float_rows(rows, cols, dtype, rows + shift)
    flat = torch.full((rows * cols + 40,), float("nan"), dtype=dtype, device=DEV)
    view = flat[shift:shift + rows * cols].view(rows, cols)
    view.copy_(x)
    q, s = ops.quantize_tokens(view)
    wq, ws = want_quantized(host(x))
    same(q, wq)
    same(s, ws)
    # q and the values in buffers with a rim of their own, rows close together
    L, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    rim = torch.full((rows * cols + 40,), 77, dtype=torch.int8, device=DEV)
    _lib.check(L.sc_quantize_tokens_device(0, view.data_ptr(), code, rows, cols, cols, rim.data_ptr() + shift, cols,
                                           s.data_ptr(), st))
    same(rim[shift:shift + rows * cols].view(rows, cols), wq)
    assert (rim[:shift] == 77).all() and (rim[shift + rows * cols:] == 77).all()
    out = torch.full((rows * cols + 40,), 5.0, dtype=dtype, device=DEV)
    for q_at, q_stride in ((q.data_ptr(), q.stride(0)), (rim.data_ptr() + shift, cols)):
        out.fill_(5.0)
        _lib.check(L.sc_dequantize_tokens_device(0, q_at, q_stride, s.data_ptr(), 0.0, rows, cols,
                                                 out.data_ptr() + shift * out.element_size(), code, cols, st))
        with np.errstate(over="ignore"):
            same(out[shift:shift + rows * cols].view(rows, cols),
                 torch.from_numpy(wq.astype(np.float32) * ws[:, None]).to(dtype).float().numpy())
        assert (out[:shift] == 5).all() and (out[shift + rows * cols:] == 5).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16, torch.int8])
@pytest.mark.parametrize("rows,k,n", [(1, 64, 33), (20, 96, 129), (700, 64, 259), (20000, 64, 131), (20001, 40, 10)])
@pytest.mark.parametrize("shift,gap", [(0, 0), (1, 0), (3, 5)])
def test_results_at_any_address(ops, dtype, rows, k, n, shift, gap):
    """Results in rows that start at any element and have a gap between them, which stays."""
    q, s = int8_rows(rows, k, 4), scales_of(rows, 5)
    w, ws, b = layer(n, k, 6)
    out = torch.full((shift + rows * (n + gap) + 9,), 5, dtype=dtype, device=DEV)
    L = _lib.load()
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int8: 3}[dtype]
    size = L.sc_int8_linear_workspace(3, 1, 1, rows, n, k, code, 0)
    work = torch.empty(max(size, 1), dtype=torch.uint8, device=DEV)
    _lib.check(L.sc_int8_linear_device(0, q.data_ptr(), 3, q.stride(0) if rows > 1 else -(-k // 16) * 16, s.data_ptr(),
                                       w.data_ptr(), w.stride(0), ws.data_ptr(), b.data_ptr(), rows, n, k, 1,
                                       out.data_ptr() + shift * out.element_size(), code, n + gap, None, 0.02,
                                       work.data_ptr() if size else None, size, torch.cuda.current_stream().cuda_stream))
    want = want_linear(host(q), host(s), host(w), host(ws), host(b), True)
    if dtype == torch.int8:
        want = np.clip(np.rint(want / np.float32(0.02)), -128, 127)
    got = out[shift:shift + rows * (n + gap)].view(rows, n + gap)
    same(got[:, :n], want)
    assert (got[:, n:] == 5).all() and (out[:shift] == 5).all() and (out[shift + rows * (n + gap):] == 5).all()


def test_wide_rows_in_a_graph(ops):
    """More channels than two accumulators hold: both launches that multiply, captured and replayed."""
    x, layers = int8_rows(6000, 96, 1), layer(1300, 96, 2)
    s = scales_of(6000, 3)
    want = ops.int8_linear_requant(x, s, *layers, relu=True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.int8_linear_requant(x, s, *layers, relu=True)
    for _ in range(3):
        got[0].zero_()
        got[1].zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_calls_from_several_threads(ops):
    """Calls of several host threads, each on a stream of its own, at the same time."""
    from concurrent.futures import ThreadPoolExecutor
    layers = [layer(512, 1024, 1), layer(900, 512, 2), layer(300, 900, 3)]
    xs = [float_rows(rows, 1024, torch.float16, rows) for rows in (1, 3, 40, 700, 3000)]
    want = [_chain(ops, x, layers, 0.02).clone() for x in xs]
    torch.cuda.synchronize()

    def work(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            out = [_chain(ops, xs[i], layers, 0.02) for _ in range(20)]
        st.synchronize()
        return all(torch.equal(o, want[i]) for o in out)

    with ThreadPoolExecutor(5) as pool:
        assert all(pool.map(work, range(5)))


def test_weights_written_right_before_the_call(ops):
    """The launch before a call writes what the call reads: weights, scales and tokens."""
    for rows in (1, 20, 3000):
        for seed in range(6):
            wf = float_rows(512, 768, torch.bfloat16, seed)
            x = float_rows(rows, 768, torch.bfloat16, seed + 50)
            w, ws = ops.quantize_tokens(wf)
            y = ops.int8_linear(x, w, ws)
            wq, wscale = want_quantized(host(wf))
            q, s = want_quantized(host(x))
            same(y, torch.from_numpy(want_linear(q, s, wq, wscale, None, False)).to(torch.bfloat16).float().numpy())


def test_no_wait_has_timed_out(ops):
    ops.check_waits(DEV)
    ops.check_waits()


def test_layer_sweep_with_token_scales():
    from sigcomp_b200.layer_sweep import token_scale_sweep
    rows = token_scale_sweep([300], repeats=2)
    assert [r[0].split(" ")[0] for r in rows] == ["layer", "hidden", "last"] and all(r[2] > 0 and r[4] > 0 for r in rows)


def test_offsets_beyond_32_bits(ops):
    """Arrays of more than 2**32 elements: their last rows come out as they do alone."""
    rows, k = 540000, 8192
    q = torch.zeros((rows, k), dtype=torch.int8, device=DEV)
    s = torch.ones(rows, device=DEV)
    tail, ts = int8_rows(300, k, 1), scales_of(300, 2)
    q[-300:], s[-300:] = tail, ts
    w, ws, b = layer(24, k, 3)
    y = ops.int8_linear(q, w, ws, b, x_scales=s)
    assert torch.equal(y[-300:], ops.int8_linear(tail, w, ws, b, x_scales=ts)) and torch.equal(y[0], b)
    x = ops.dequantize_tokens(q, s, dtype=torch.bfloat16)
    del q
    assert torch.equal(x[-300:], ops.dequantize_tokens(tail, ts, dtype=torch.bfloat16)) and not x[-301].any()
    again, scales = ops.quantize_tokens(x)
    want, wscales = ops.quantize_tokens(x[-300:])
    assert torch.equal(again[-300:], want) and torch.equal(scales[-300:], wscales) and not again[-301].any()


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("rows,n", [(3, 40), (70, 512), (6000, 300), (6000, 512), (6000, 900)])
def test_requantised_rows_of_extreme_results(ops, relu, rows, n):
    """Results far below zero, infinite or NaN through the bias, and rows that ReLU leaves empty."""
    q, s = int8_rows(rows, 64, 1), scales_of(rows, 2)
    w, ws, _ = layer(n, 64, 3)
    for value in (-1e30, float("-inf"), float("inf"), float("nan"), -1.0):
        b = torch.zeros(n, device=DEV) if value != -1.0 else torch.full((n,), -50.0, device=DEV)
        b[n // 2] = value
        with np.errstate(invalid="ignore", over="ignore"):
            y = want_linear(host(q), host(s), host(w), host(ws), host(b), relu)
        wq, wscale = want_quantized(y)
        yq, ys = ops.int8_linear_requant(q, s, w, ws, b, relu=relu)
        same(ys, wscale)
        same(yq, wq)


@pytest.mark.parametrize("rows", [1, 20, 6000])
@pytest.mark.parametrize("scale", [0.06, 1.0, 0.011, 3.7, 2.0 ** -120, 3e30, 1.1e-38])
@pytest.mark.parametrize("relu", [False, True])
def test_logits_next_to_a_half(ops, rows, scale, relu):
    """Results at halves of the output scale, next to them on both sides, beyond the ends, and no numbers."""
    scale32 = np.float32(scale)
    half = (np.arange(-131, 131, dtype=np.float64) + 0.5) * np.float64(scale32)
    with np.errstate(over="ignore"):
        at = half.astype(np.float32)
        values = np.concatenate([np.nextafter(at, np.float32(-np.inf)), at, np.nextafter(at, np.float32(np.inf)),
                                 np.float32([np.nan, np.inf, -np.inf, 0, -0.0, 1e38, -1e38, 1e-40, -1e-45])])
    n = len(values)
    q, s = torch.zeros((rows, 64), dtype=torch.int8, device=DEV), torch.ones(rows, device=DEV)
    w, ws, _ = layer(n, 64, 3)
    got = ops.int8_linear_requant(q, s, w, ws, torch.from_numpy(values).to(DEV), relu=relu, output_scale=float(scale32))
    y = np.where(values < 0, np.float32(0), values) if relu else values
    with np.errstate(over="ignore", invalid="ignore"):
        want = np.clip(np.rint(y / scale32), -128, 127)
    want = np.where(np.isnan(want), 0, want).astype(np.int8)
    same(got, np.tile(want, (rows, 1)))
