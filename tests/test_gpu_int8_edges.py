"""The int8 operators on a GPU at calls that their first tests leave out, against the same definition."""

import threading
import time

import numpy as np
import pytest
import torch

from test_gpu_int8 import DEV, host, layer, same, want_linear, want_quantized

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from sigcomp_b200 import int8
    return int8


# ---- infinite scales ---------------------------------------------------------------------------

@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("k,n", [(64, 1), (64, 33), (64, 40), (512, 130), (512, 300), (96, 500), (96, 900), (64, 512)])
def test_infinite_scales_of_rows(ops, k, n, relu):
    """Rows whose scale is infinite: sums below zero are minus infinity, which ReLU makes 0, so the row can be
    quantised; sums above zero and sums of zero (a NaN) make it one that cannot be.  The same in a batch of any size."""
    kinds = 6
    q = torch.zeros((kinds, k), dtype=torch.int8, device=DEV)
    q[0], q[1], q[2, 0], q[4], q[5] = 1, -1, 0, 1, 100          # row 2: sums of zero; 3: an ordinary row of zeros
    s = torch.tensor([np.inf, np.inf, np.inf, 1.0, -np.inf, 0.5], device=DEV)
    w = torch.full((n, -(-k // 16) * 16), -1, dtype=torch.int8, device=DEV)[:, :k]
    w[n // 2] = -3
    _, ws, b = layer(n, k, 3)
    with np.errstate(invalid="ignore", over="ignore"):
        y = want_linear(host(q), host(s), host(w), host(ws), host(b), relu)
    wq, wscale = want_quantized(y)
    assert np.isfinite(wscale[0]) == relu and np.isnan(wscale[1:3]).all()
    for rows in (1, 2, 3, 6, 40, 700, 6000, 20000):
        pick = torch.arange(rows, device=DEV) % kinds
        idx = pick.cpu().numpy()
        yq, ys = ops.int8_linear_requant(q[pick], s[pick], w, ws, b, relu=relu)
        same(ys, wscale[idx])
        same(yq, wq[idx])
        same(ops.int8_linear(q[pick], w, ws, b, x_scales=s[pick], relu=relu), y[idx])


# ---- derivatives and batching by torch ---------------------------------------------------------

def test_tangents_and_transforms_are_refused(ops):
    """A dual tensor's tangent would be lost, and a batched one has no memory of its own."""
    x, (w, ws, b) = torch.randn(4, 64, device=DEV), layer(32, 64, 1)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match="derivative"):
            ops.int8_linear(dual, w, ws, b)
        assert torch.equal(ops.int8_linear(torch.autograd.forward_ad.unpack_dual(dual).primal, w, ws, b),
                           ops.int8_linear(x, w, ws, b))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v: ops.int8_linear(v, w, ws, b))(x)
    for transform in (torch.func.grad, torch.func.jacfwd):
        with pytest.raises(ValueError, match="gradient|derivative"):
            transform(lambda v: ops.int8_linear(v, w, ws, b).sum())(x)


# ---- host side ---------------------------------------------------------------------------------

def test_other_threads_run_while_a_call_waits_for_the_stream(ops):
    """More launches than the driver queues, behind work of about a second: the call that has to wait for room lets
    the process's other Python threads run."""
    x, (w, ws, b) = torch.randn(4, 64, device=DEV), layer(32, 64, 1)
    ops.int8_linear(x, w, ws, b)
    torch.cuda.synchronize()
    beats, stop = [], threading.Event()

    def beat():
        while not stop.is_set():
            beats.append(time.perf_counter())
            time.sleep(0.005)

    thread = threading.Thread(target=beat)
    thread.start()
    try:
        torch.cuda._sleep(2_000_000_000)
        longest = 0.0
        for _ in range(3000):
            t = time.perf_counter()
            ops.int8_linear(x, w, ws, b)
            longest = max(longest, time.perf_counter() - t)
        torch.cuda.synchronize()
    finally:
        stop.set()
        thread.join()
    assert longest > 0.3, "no call had to wait: the test shows nothing"
    assert np.diff(beats).max() < 0.25


def test_check_of_waits_is_refused_during_a_capture(ops):
    """It has to wait for the stream, which a capture cannot; the refusal leaves the capture as it is."""
    x, (w, ws, b) = torch.randn(20, 64, device=DEV), layer(32, 64, 1)
    want = ops.int8_linear(x, w, ws, b)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.int8_linear(x, w, ws, b)
        with pytest.raises(ValueError, match="captured"):
            ops.check_waits()
    got.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    ops.check_waits()


def test_capture_over_two_streams(ops):
    """Operators on a stream that a capture forks to, and one that reads the results of both after the join."""
    x = torch.randn(300, 512, device=DEV)
    a, b, last = layer(512, 512, 1), layer(512, 512, 2), layer(96, 512, 3)

    def run(side):
        main = torch.cuda.current_stream()
        q, s = ops.quantize_tokens(x)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            right = ops.int8_linear_requant(q, s, *b, relu=True)
        left = ops.int8_linear_requant(q, s, *a, relu=True)
        main.wait_stream(side)
        return ops.int8_linear(left[0], *last, x_scales=left[1]), ops.int8_linear(right[0], *last, x_scales=right[1])

    side = torch.cuda.Stream()
    want = [t.clone() for t in run(side)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run(side)
    for _ in range(3):
        for t in got:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t, v) for t, v in zip(got, want))


# ---- waits that give up ------------------------------------------------------------------------

def test_a_wait_that_gives_up_is_reported_to_every_thread(ops):
    """A kernel whose wait nothing ends gives up after its limit.  Each thread's next check raises, once, whichever
    thread asks first, and the operators work as before."""
    from sigcomp_b200 import _lib

    def check():
        try:
            ops.check_waits()
        except _lib.CodecError as e:
            return "timed out" in str(e)
        return False

    ask, answers = threading.Barrier(2, timeout=60), []

    def other():
        torch.cuda.set_device(0)
        check()                          # what was before
        ask.wait()
        ask.wait()
        answers.append(check())
        answers.append(check())

    thread = threading.Thread(target=other)
    thread.start()
    check()
    ask.wait()
    _lib.check(_lib.load().sc_selftest_int8_wait_timeout(0, torch.cuda.current_stream().cuda_stream))
    assert check() and not check()
    ask.wait()
    thread.join()
    assert answers == [True, False]
    x, (w, ws, b) = torch.randn(3000, 512, device=DEV), layer(512, 512, 1)
    q, s = want_quantized(host(x))
    same(ops.int8_linear(x, w, ws, b), want_linear(q, s, host(w), host(ws), host(b), False))
    assert not check()


# ---- errors of the CUDA runtime ----------------------------------------------------------------

def test_a_failed_call_leaves_no_error_behind(ops):
    """The runtime keeps a failed call's error for the thread until someone asks for it.  Torch asks after each of its
    launches, so an error that is returned as a status must not be left for it."""
    import ctypes
    from sigcomp_b200 import _lib
    L = _lib.load()
    runtime = next(line.split()[-1] for line in open("/proc/self/maps") if "libcudart" in line)
    last = ctypes.CDLL(runtime).cudaGetLastError
    last()
    some = 4096                                                # not read: there is no device 9999
    assert L.sc_quantize_tokens_device(9999, some, 0, 4, 8, 8, some, 8, some, None) == _lib.SC_ERR_CUDA
    assert last() == 0
    assert L.sc_int8_status_device(9999, None) == _lib.SC_ERR_CUDA
    assert last() == 0
    x = torch.ones(8, device=DEV)
    assert torch.cuda.current_device() == 0 and (x + 1).sum().item() == 16


# ---- decoding ----------------------------------------------------------------------------------

def test_decoding_step_by_step(ops):
    """A model whose next logits depend on the symbols decoded before: each step computes one row of logits per stream,
    from the decoded symbols alone, and decodes the streams' prefixes with the rows so far."""
    import ctypes
    from sigcomp_b200 import _lib
    from sigcomp_b200.codec import B200Compression
    from sigcomp_b200.model import random_model
    model = random_model(3)
    codec = B200Compression(chunk_len=2048, gpu=0, model=model)
    streams, steps, window = 5, 24, model.window_size
    table = torch.from_numpy(model.embedding.astype(np.float32)).to(torch.bfloat16).to(DEV)
    layers = [layer(512, window * model.emb_dim, 1), layer(512, 512, 2), layer(256, 512, 3)]
    scale = float(model.output_scale)
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    p = lambda t: ctypes.c_void_p(t.data_ptr())

    def logits_of(ids):
        q, s = ops.quantize_tokens(table[ids].flatten(-2))
        for l in layers[:-1]:
            q, s = ops.int8_linear_requant(q, s, *l, relu=True)
        return ops.int8_linear_requant(q, s, *layers[-1], output_scale=scale)

    symbols = np.random.default_rng(1).integers(0, 256, size=(streams, steps)).astype(np.uint8)
    sym = torch.from_numpy(symbols).to(DEV)
    known = torch.cat([torch.full((streams, window), 256, device=DEV), sym.long()], dim=1)
    batch = logits_of(known.unfold(1, window, 1)[:, :steps]).contiguous()
    off = torch.arange(0, streams * steps + 1, steps, dtype=torch.int64, device=DEV)
    words = torch.zeros(streams * (steps + 2), dtype=torch.int32, device=DEV)
    woff = torch.zeros(streams + 1, dtype=torch.int64, device=DEV)
    _lib.check(codec._lib.sc_encode_logits_device(codec.handle, p(batch), p(sym.contiguous()), p(off), streams, p(words),
                                                  words.numel(), p(woff), None, st))
    context = torch.full((streams, window), 256, device=DEV)
    rows, back = [], None
    for t in range(steps):
        rows.append(logits_of(context))
        so_far = torch.stack(rows, dim=1).contiguous()
        back = torch.zeros((streams, t + 1), dtype=torch.uint8, device=DEV)
        off = torch.arange(0, streams * (t + 1) + 1, t + 1, dtype=torch.int64, device=DEV)
        _lib.check(codec._lib.sc_decode_logits_device(codec.handle, p(so_far), p(off), p(words), p(woff), streams, p(back),
                                                      None, st))
        context = torch.cat([context[:, 1:], back[:, t:].long()], dim=1)
    assert torch.equal(back, sym)
    codec.close()


def test_a_result_that_does_not_fit_is_a_memory_error(ops):
    """The allocation fails while Python's lock is released: the error is raised all the same, and calls work after it."""
    rows = 2_000_000_000
    q, s = torch.ones((1, 16), dtype=torch.int8, device=DEV), torch.ones(1, device=DEV)
    w, ws, b = layer(64, 16, 1)
    want = ops.int8_linear(q, w, ws, b, x_scales=s)
    with pytest.raises(MemoryError):
        ops.int8_linear(q.expand(rows, 16), w, ws, b, x_scales=s.expand(rows))             # 512 GB
    with pytest.raises(MemoryError):
        ops.dequantize_tokens(q.expand(3 * rows, 16), 1.0)
    assert torch.equal(ops.int8_linear(q, w, ws, b, x_scales=s), want)
