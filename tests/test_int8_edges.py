"""Refusals of the int8 operators that need no GPU, beyond the plain ones."""

import pytest
import torch
from torch.autograd import forward_ad

from sigcomp_b200.int8 import dequantize_tokens, int8_linear, int8_linear_requant, quantize_tokens

X = torch.zeros((4, 32))
Q = torch.zeros((4, 32), dtype=torch.int8)
S = torch.ones(4)
W = torch.zeros((8, 32), dtype=torch.int8)
T = torch.ones(8)
B = torch.zeros(8)


# ---- forward-mode derivatives ------------------------------------------------------------------

CALLS = {
    "quantize": (X, lambda d: quantize_tokens(d)),
    "dequantize scales": (S, lambda d: dequantize_tokens(Q, d)),
    "linear x": (X, lambda d: int8_linear(d, W, T, B)),
    "linear weight_scales": (T, lambda d: int8_linear(X, W, d, B)),
    "linear bias": (B, lambda d: int8_linear(X, W, T, d)),
    "linear x_scales": (S, lambda d: int8_linear(Q, W, T, B, x_scales=d)),
    "requant scales": (S, lambda d: int8_linear_requant(Q, d, W, T)),
    "requant bias": (B, lambda d: int8_linear_requant(Q, S, W, T, d)),
}


@pytest.mark.parametrize("name", CALLS)
def test_tangents_are_refused(name):
    """A dual tensor asks for a derivative in the forward direction, also where no gradient is recorded."""
    primal, call = CALLS[name]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(primal, torch.ones_like(primal))
        with pytest.raises(ValueError, match="derivative"):
            call(dual)
        with torch.no_grad(), pytest.raises(ValueError, match="derivative"):
            call(dual)
        with pytest.raises(ValueError, match="run on a GPU"):
            call(forward_ad.unpack_dual(dual).primal)


@pytest.mark.parametrize("transform", [
    lambda f: torch.func.jvp(f, (X,), (torch.ones_like(X),)), lambda f: torch.func.grad(f)(X),
    lambda f: torch.func.jacfwd(f)(X), lambda f: torch.func.jacrev(f)(X),
])
def test_derivatives_by_function_transforms_are_refused(transform):
    with pytest.raises((ValueError, RuntimeError), match="derivative|gradient|storage"):
        transform(lambda x: int8_linear(x, W, T).sum())


# ---- build -------------------------------------------------------------------------------------

def test_build_refuses_spills_in_the_kernels_that_load_tensor_memory():
    """Both int8 kernels read TMEM into registers asynchronously: neither may spill."""
    import re
    from sigcomp_b200 import build_ext
    loading = set()
    for name in ("sc_int8.cu", "sc_int8_mm.cuh", "sc_int8_token.cuh"):
        parts = re.split(r"__global__", (build_ext.CSRC / name).read_text())[1:]
        loading |= {re.search(r"\b(k_\w+)\(", p).group(1) for p in parts if "tmem_ld" in p}
    assert loading == {"k_pair", "k_few"}
    assert loading <= set(build_ext.NO_SPILL_KERNELS) and "sc_int8.cu" in build_ext.NO_SPILL_SOURCES


def test_binding_of_another_torch_is_rebuilt_and_not_used(monkeypatch, tmp_path):
    """The binding is compiled against torch's headers: another version of torch makes it stale."""
    import subprocess
    import sys
    from sigcomp_b200 import build_ext
    done = subprocess.run([sys.executable, "-c", "import torch; torch.__version__ = '9.9.0'; import sigcomp_b200.int8"],
                          cwd=build_ext.PKG.parent, capture_output=True, text=True)
    assert done.returncode != 0 and "was built for torch" in done.stderr
    monkeypatch.setattr(build_ext, "BINDING", tmp_path / "_int8.so")
    monkeypatch.setattr(build_ext, "BINDING_STAMP", tmp_path / "stamp")
    build_ext.BINDING.write_bytes(b"")
    assert build_ext._binding_stale()                      # built for an unknown torch
    build_ext.BINDING_STAMP.write_text(build_ext._built_for())
    assert not build_ext._binding_stale()
    monkeypatch.setattr(torch, "__version__", "9.9.0")
    assert build_ext._binding_stale()


# ---- the ways of a call ------------------------------------------------------------------------

def _ways(rows, k, n, scaled):
    """((rows, kernel, tile, split, ns), ...) of a call's parts."""
    import ctypes
    from sigcomp_b200 import _lib
    out = (ctypes.c_int64 * 10)()
    parts = _lib.load().sc_int8_linear_ways(rows, n, k, scaled, out)
    return tuple(tuple(out[5 * i:5 * i + 5]) for i in range(parts))


def test_ways_hold_all_rows():
    for scaled in (0, 1):
        for shape in ((1, 1, 1), (20480, 8192, 512), (9473, 2048, 300), (2 ** 31 - 1025, 1, 1)):
            ways = _ways(*shape, scaled)
            assert sum(w[0] for w in ways) == shape[0] and all(w[0] > 0 and w[4] > 0 for w in ways)
    for shape in ((0, 8, 8), (-1, 8, 8), (8, 0, 8), (8, 8, 0), (8, 131072, 8), (2 ** 31, 8, 8)):
        assert _ways(*shape, 1) == ()


def test_tested_shapes_reach_every_way():
    """Kernels, tiles and cuts that the sizes of a wide grid choose are all reached by the shapes that the GPU tests compare
    with the definition."""
    import test_gpu_int8
    import test_gpu_int8_ways
    tested = test_gpu_int8.SIZES + test_gpu_int8_ways.WHOLE + test_gpu_int8_ways.CUT

    def kinds(shapes):
        return {(scaled,) + tuple(w[1:3] for w in _ways(*shape, scaled)) for shape in shapes for scaled in (0, 1)}

    grid = [(rows, k, n) for rows in (1, 2, 3, 8, 20, 60, 200, 1000, 3000, 9473, 10000, 18945, 19000, 19200, 20480, 38000, 40000)
            for k in (64, 512, 2048, 4096, 8192) for n in (8, 96, 256, 300, 512, 700, 1300, 2304, 4096)]
    assert kinds(grid) - kinds(tested) == set()
    # K of k_few's tiles split in every number of parts
    splits = {w[2:4] for shape in tested for scaled in (0, 1) for w in _ways(*shape, scaled) if w[1] == 1}
    assert splits >= {w[2:4] for shape in grid for scaled in (0, 1) for w in _ways(*shape, scaled) if w[1] == 1}
