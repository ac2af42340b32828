"""Refusals of the 8-bit saved activations that need no GPU: the library's entry points check
their arguments before any HIP call, the Python layer refuses tensors that are not on a GPU."""
import ctypes

import pytest
import torch


def _lib():
    from sgnn_amd import _lib
    return _lib, _lib.load()


P = ctypes.c_void_p(4096)                            # never followed: every call below is refused


@pytest.mark.parametrize("dtype,n,F,ldx,slope,x,codes,word", [
    (2, 4, 8, 8, 1.0, P, P, b"type"), (0, -1, 8, 8, 1.0, P, P, b"n >= 0"), (0, 4, 0, 8, 1.0, P, P, b"F > 0"),
    (0, 4, 8, 7, 1.0, P, P, b"stride"), (0, 4, 8, 8, -0.5, P, P, b"slope"), (0, 4, 8, 8, float("nan"), P, P, b"slope"),
    (0, 4, 8, 8, float("inf"), P, P, b"slope"), (1, 4, 8, 8, 1.0, None, P, b"null"), (1, 4, 8, 8, 1.0, P, None, b"null"),
    (1, 4, 8, 8, 1.0, P, ctypes.c_void_p(4097), b"aligned"), (0, 4, 1 << 30, 1 << 30, 1.0, P, P, b"features"),
])
def test_save_refuses(dtype, n, F, ldx, slope, x, codes, word):
    mod, lib = _lib()
    rc = lib.sgnn_save8(dtype, n, F, x, ldx, slope, codes, P, None)
    assert rc < 0 and word in lib.sgnn_last_error()
    with pytest.raises(mod.SgnnHipError):
        mod.check(rc)


def test_the_other_entry_points_refuse():
    _, lib = _lib()
    assert lib.sgnn_saved8_linear(0, 4, 8, 0, P, 8, P, 8, 0.0, P, P, P, 4, None) == -1
    assert lib.sgnn_saved8_linear(0, 4, 8, 4, P, 7, P, 8, 0.0, P, P, P, 4, None) == -1
    assert lib.sgnn_saved8_linear(0, 4, 8, 4, P, 8, P, 7, 0.0, P, P, P, 4, None) == -1
    assert lib.sgnn_saved8_linear(0, 4, 8, 4, P, 8, P, 8, 0.0, P, P, P, 3, None) == -1
    assert lib.sgnn_saved8_linear(0, 4, 8, 4, P, 8, P, 8, 0.0, P, None, P, 4, None) == -1
    assert lib.sgnn_saved8_linear(0, 4, 8, 4, P, 8, None, 8, 0.0, P, P, P, 4, None) == -1
    assert lib.sgnn_saved8_linear(3, 4, 8, 4, P, 8, P, 8, 0.0, P, P, P, 4, None) == -1
    assert lib.sgnn_saved8_linear_grad(0, 4, 8, 4, None, 0.0, P, 4, P, 8, P, 8, None) == -1
    assert lib.sgnn_saved8_linear_grad(0, 4, 8, 4, P, 0.0, P, 3, P, 8, P, 8, None) == -1
    assert lib.sgnn_saved8_linear_grad(0, 4, 8, 4, P, 0.0, P, 4, P, 8, P, 7, None) == -1
    assert lib.sgnn_restore8(0, 4, 8, P, P, 0.0, P, 7, None) == -1
    assert lib.sgnn_restore8(0, 4, 8, P, None, 0.0, P, 8, None) == -1
    assert lib.sgnn_saved8_input_grad(0, 4, 8, P, 1.0, P, 8, P, 8, None) == -1
    assert lib.sgnn_saved8_input_grad(0, 4, 8, P, 0.0, P, 7, P, 8, None) == -1
    assert lib.sgnn_saved8_input_grad(0, 4, 8, P, 0.0, None, 8, P, 8, None) == -1
    need = lib.sgnn_saved8_weight_grad_workspace_bytes(100_000, 64, 32)
    assert need > 0 and lib.sgnn_saved8_weight_grad_workspace_bytes(0, 64, 32) == 0
    assert lib.sgnn_saved8_weight_grad(0, 100_000, 64, 32, P, P, 0.0, P, 32, P, 64, P, need - 1, None) == -2
    assert lib.sgnn_saved8_weight_grad(0, 100_000, 64, 32, P, P, 0.0, P, 32, P, 64, None, need, None) == -1
    assert lib.sgnn_saved8_weight_grad(0, 100_000, 64, 32, P, P, 0.0, P, 31, P, 64, P, need, None) == -1
    assert lib.sgnn_saved8_weight_grad(0, 100_000, 64, 32, P, P, 0.0, P, 32, P, 63, P, need, None) == -1
    assert lib.sgnn_saved8_weight_grad(0, 0, 64, 32, P, P, 0.0, P, 32, P, 64, P, need, None) == -1
    assert lib.sgnn_saved8_weight_grad(0, 100_000, 64, 0, P, P, 0.0, P, 32, P, 64, P, need, None) == -1


def test_nothing_to_do_is_not_an_error():
    _, lib = _lib()
    assert lib.sgnn_save8(0, 0, 8, None, 8, 0.0, None, None, None) == 0
    assert lib.sgnn_saved8_linear(0, 0, 8, 4, None, 8, None, 8, 0.0, None, None, None, 4, None) == 0
    assert lib.sgnn_saved8_linear_grad(0, 0, 8, 4, None, 0.0, None, 4, None, 8, None, 8, None) == 0
    assert lib.sgnn_restore8(1, 0, 8, None, None, 0.0, None, 8, None) == 0
    assert lib.sgnn_saved8_input_grad(1, 0, 8, None, 0.0, None, 8, None, 8, None) == 0


def test_python_layer_needs_gpu_tensors():
    from sgnn_amd import nn
    x = torch.randn(4, 8)
    with pytest.raises(ValueError):
        nn.save_int8(x)
    with pytest.raises(ValueError):
        nn.linear_saved_int8(x, torch.randn(2, 8))
    with pytest.raises(ValueError):
        nn.SavedInt8(torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.uint8), (4, 8), 0.0,
                     torch.float32)
