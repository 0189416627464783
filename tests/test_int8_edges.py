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
