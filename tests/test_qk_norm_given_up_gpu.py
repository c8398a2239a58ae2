"""Gradients of a norm whose kernels have given up: the weights' gradients are NaN, never sums of what there was.

Once a bounded wait has run out, later launches of these kernels do nothing, and the sticky word says so.  No test makes a wait run out: the word is
set from the host, in a copy of the kernels compiled here for that, whose word is its own."""
import ctypes
import pathlib
import shutil
import subprocess

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CSRC = pathlib.Path(__file__).resolve().parent.parent / "dashmag_b200" / "csrc"
SOURCE = """
#include "%s/qk_norm.cu"
extern "C" int set_word(unsigned int x) { return (int)cudaMemcpyToSymbol(dash::g_qk_norm_status, &x, sizeof x); }
extern "C" int backward(const void *x, const void *g, const void *w, void *dx, void *dw, const void *cos, const void *sin, float *part, long long tokens, int heads, int d) {
    dash::NormArgs a{};
    a.q = dash::NormTensor{x, 0, (long long)heads * d, d, g, 0, (long long)heads * d, d, dx, w, dw, heads};
    a.b = 1; a.t = tokens; a.d = a.dim = d; a.eps = 1e-6f;
    a.cos = cos; a.sin = sin; a.len = tokens; a.part = part;
    int launches = 0;
    return (int)dash::launch_qk_norm_backward(1, a, nullptr, &launches);
}
extern "C" unsigned long long part_floats(int d) { return dash::qk_norm_part_floats(d); }
"""


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not pathlib.Path(nvcc).exists():
        pytest.skip("no nvcc")
    at = tmp_path_factory.mktemp("kernels")
    (at / "words.cu").write_text(SOURCE % CSRC)
    done = subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-split-compile=0", "-Xptxas", "-O1", "-std=c++17", "-Xcompiler", "-fPIC",
                           "--expt-relaxed-constexpr", "-shared", "-cudart", "static", "-o", str(at / "words.so"), str(at / "words.cu")],
                          capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stderr
    lib = ctypes.CDLL(str(at / "words.so"))
    lib.part_floats.restype = ctypes.c_ulonglong
    return lib


@pytest.mark.parametrize("tokens,heads,d", [(3, 2, 64), (5000, 8, 128)])
def test_the_weights_gradient(kernels, tokens, heads, d):
    randn = lambda *shape: torch.randn(*shape, dtype=torch.bfloat16, device=DEV)
    x, g, w = randn(tokens, heads, d), randn(tokens, heads, d), randn(d)
    dx, dw = torch.empty_like(x), torch.zeros_like(w)
    cos, sin = torch.ones(tokens, d, dtype=torch.bfloat16, device=DEV), torch.zeros(tokens, d, dtype=torch.bfloat16, device=DEV)
    part = torch.empty(kernels.part_floats(d), device=DEV)
    pointer = lambda t: ctypes.c_void_p(t.data_ptr())

    def backward():
        torch.cuda.synchronize()   # (the call is on the default stream of another runtime)
        assert kernels.backward(*map(pointer, (x, g, w, dx, dw, cos, sin, part)), ctypes.c_longlong(tokens), heads, d) == 0
        torch.cuda.synchronize()
        return dw.double()

    x64 = x.double()
    want = (g.double() * x64 / torch.sqrt(x64.square().mean(-1, keepdim=True) + 1e-6)).sum((0, 1))
    size = (g.double() * x64 / torch.sqrt(x64.square().mean(-1, keepdim=True) + 1e-6)).abs().sum((0, 1))
    within = lambda got: bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 300 * 2.0 ** -24 * size).all())   # the dtype's half step, the sums' as in the operator's tests
    assert within(backward())
    try:
        assert kernels.set_word(16) == 0
        assert bool(torch.isnan(backward()).all())
    finally:
        assert kernels.set_word(0) == 0
    assert within(backward())
