"""The layers in front of the document head, without a GPU: refusals, argument checks of the C entry points, struct layout."""

import ctypes as C
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def layers():
    from late_interaction_kernels_b200 import _build, token_layers

    _build.build()
    return token_layers


def test_no_cpu_path(layers):
    x, w = torch.zeros(2, 8), torch.zeros(8, 8)
    for fn in (lambda: layers.layer_norm(x), lambda: layers.linear(x, w), lambda: layers.gated_feed_forward(x, w, w, w)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            fn()


def test_struct_sizes_are_the_compilers(layers, tmp_path):
    from late_interaction_kernels_b200 import _lib

    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "lik_b200.h"\nint main(void) { printf("%zu %zu %zu", sizeof(lik_norm_args), sizeof(lik_linear_args), '
                   "sizeof(lik_gated_args)); return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    out = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout
    assert out == " ".join(str(C.sizeof(t)) for t in (_lib.NormArgs, _lib.LinearArgs, _lib.GatedArgs))


def test_c_entries_refuse_before_any_launch(layers):
    from late_interaction_kernels_b200 import _lib

    lib = _lib.load()
    for name, args in (("layer_norm", _lib.NormArgs), ("linear", _lib.LinearArgs), ("gated", _lib.GatedArgs)):
        for way in ("fwd", "bwd"):
            fn = getattr(lib, f"lik_{name}_{way}")
            assert fn(None, None) == -1
            a = args()
            a.dtype = a.param_dtype = _lib.LIK_BF16
            assert fn(C.byref(a), None) == -1 and b"positive" in lib.lik_last_error()
            a.dtype = _lib.LIK_E4M3
            assert fn(C.byref(a), None) == -1 and b"dtype must be" in lib.lik_last_error()
    a = _lib.LinearArgs(dtype=2, param_dtype=2, x_stride=8, w_stride=8, rows=4, out=8, activation=9)
    setattr(a, "in", 8)
    assert lib.lik_linear_fwd(C.byref(a), None) == -1 and b"activation" in lib.lik_last_error()
    a.activation = 3
    assert lib.lik_linear_fwd(C.byref(a), None) == -1 and b"must not be NULL" in lib.lik_last_error()
    a.param_dtype = _lib.LIK_F16
    assert lib.lik_linear_bwd(C.byref(a), None) == -1 and b"param_dtype" in lib.lik_last_error()
    n = _lib.NormArgs(dtype=2, param_dtype=0, x_stride=8, rows=4, width=8, eps=-1.0)
    assert lib.lik_layer_norm_fwd(C.byref(n), None) == -1 and b"eps" in lib.lik_last_error()


def test_workspace_queries_need_no_gpu(layers):
    """A serving runtime plans its memory ahead: sizes come from the arguments alone, and a larger call needs no less."""
    from late_interaction_kernels_b200 import _lib

    lib = _lib.load()

    def linear(rows, dtype, odd=0):
        a = _lib.LinearArgs(x=4096, w=4096, dy=4096, dx=4096, dw=4096, dbias=4096, z=4096, x_stride=768 + odd, w_stride=768 + odd, dy_stride=512, z_stride=512,
                            rows=rows, out=512, dtype=dtype, param_dtype=dtype, activation=3)
        setattr(a, "in", 768)
        return lib.lik_linear_fwd_workspace(C.byref(a)), lib.lik_linear_bwd_workspace(C.byref(a))

    def gated(rows, dtype):
        a = _lib.GatedArgs(x=4096, w_gate=4096, w_up=8192, w_down=16384, dy=4096, dx=4096, dw_gate=4096, dw_up=4096, dw_down=4096, db_gate=4096, db_up=4096, db_down=4096,
                           x_stride=768, w_gate_stride=768, w_up_stride=768, w_down_stride=1100, dy_stride=768, kept_stride=1104, rows=rows, hidden=1100, out=768,
                           dtype=dtype, param_dtype=dtype, activation=2)
        setattr(a, "in", 768)
        return lib.lik_gated_fwd_workspace(C.byref(a)), lib.lik_gated_bwd_workspace(C.byref(a))

    for fn in (linear, gated):
        for dtype in (_lib.LIK_BF16, _lib.LIK_F16, _lib.LIK_F32):
            assert fn(0, dtype) == (0, 0)
            sizes = [fn(rows, dtype) for rows in (1, 100, 100_000, 2_000_000_000)]
            for small, large in zip(sizes, sizes[2:]):
                assert small[0] <= large[0] and small[1] < large[1]
    # rows that TMA cannot address ask for room for a copy
    assert linear(5000, _lib.LIK_BF16, odd=1)[0] >= 5000 * 768 * 2 > linear(5000, _lib.LIK_BF16)[0]
    a = _lib.NormArgs(dtype=2, param_dtype=2, x_stride=768, rows=10**9, width=768, dweight=4096, eps=1e-5)
    assert 0 < lib.lik_layer_norm_bwd_workspace(C.byref(a)) < 16 << 20


def test_a_kept_side_of_relu_asks_for_workspace_and_says_so(layers):
    """relu's forward pass takes its rows' lengths first where a backward pass follows: a call without the room for them is refused before any launch."""
    from late_interaction_kernels_b200 import _lib

    lib = _lib.load()
    for rows in (3, 5000):
        a = _lib.LinearArgs(x=4096, w=4096, y=4096, x_stride=768, w_stride=768, z_stride=512, rows=rows, out=512, dtype=_lib.LIK_BF16, param_dtype=_lib.LIK_BF16, activation=1)
        setattr(a, "in", 768)
        without = lib.lik_linear_fwd_workspace(C.byref(a))
        a.z = 4096
        assert lib.lik_linear_fwd_workspace(C.byref(a)) >= without + 4 * (rows + 512)
        a.workspace_bytes = without
        assert lib.lik_linear_fwd(C.byref(a), None) != 0 and b"workspace" in lib.lik_last_error()
        a.activation = 3
        assert lib.lik_linear_fwd_workspace(C.byref(a)) == without


def test_only_what_is_made_of_dy_needs_nothing_kept(layers):
    from late_interaction_kernels_b200 import _lib

    lib = _lib.load()
    a = _lib.GatedArgs(x=4096, w_gate=4096, w_up=8192, w_down=16384, dy=4096, db_down=4096, x_stride=64, w_gate_stride=64, w_up_stride=64, w_down_stride=128, dy_stride=64,
                       rows=300, hidden=128, out=64, dtype=_lib.LIK_BF16, param_dtype=_lib.LIK_BF16, activation=2)
    setattr(a, "in", 64)
    assert lib.lik_gated_bwd(C.byref(a), None) != 0 and b"workspace" in lib.lik_last_error()  # (past the check of what is kept)
    a.dw_down = 4096
    assert lib.lik_gated_bwd(C.byref(a), None) == -1 and b"must be there" in lib.lik_last_error()
