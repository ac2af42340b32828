"""Refusals of the class cross-entropy that need no GPU."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(4096)                            # never followed: every call below is refused
BIG = 1 << 40


def _lib():
    from sgnn_amd import _lib
    return _lib.load()


def forward(lib, dtype=0, B=10, D=8, V=70, x=P, ldx=8, w=P, sv=8, sd=1, labels=P, n=10, idx=None, stats=P, rows=P,
            loss=P, share=P, ws=P, ws_bytes=BIG):
    return lib.sgnn_class_xent_forward(dtype, B, D, V, x, ldx, w, sv, sd, labels, n, idx, stats, rows, loss, share, ws,
                                       ws_bytes, None)


def backward(lib, dx=P, lddx=8, dw=P, dsv=8, dsd=1, grad=P, stats=P, ws=P, ws_bytes=BIG, B=10, ldx=8):
    return lib.sgnn_class_xent_backward(0, B, 8, 70, P, ldx, P, 8, 1, P, 10, None, stats, grad, None, dx, lddx, dw, dsv,
                                        dsd, ws, ws_bytes, None)


@pytest.mark.parametrize("bad,rc,word", [
    (dict(dtype=2), -1, b"type"), (dict(B=0), -1, b"B > 0"), (dict(V=-1), -1, b"V > 0"), (dict(D=0), -1, b"D > 0"),
    (dict(ldx=7), -1, b"stride"), (dict(sv=7), -1, b"unit stride"), (dict(sv=16, sd=2), -1, b"unit stride"),
    (dict(sv=1, sd=69), -1, b"unit stride"), (dict(n=9), -1, b"labels"), (dict(n=-1, idx=P), -1, b"labels"),
    (dict(x=None), -1, b"null"), (dict(w=None), -1, b"null"), (dict(labels=None), -1, b"null"),
    (dict(stats=None), -1, b"null"), (dict(rows=None), -1, b"null"), (dict(share=None), -1, b"null"),
    (dict(ws=None), -1, b"null"), (dict(ws_bytes=16), -2, b"workspace"), (dict(V=1 << 29), -4, b"2^28"),
    (dict(B=1 << 26, n=1 << 26), -4, b"2^25"), (dict(V=1 << 28, D=65, ldx=65, sv=65), -4, b"2^33"),
    (dict(D=1 << 17, ldx=1 << 17, sv=1 << 17), -4, b"65536"),
])
def test_forward_refuses(bad, rc, word):
    lib = _lib()
    assert forward(lib, **bad) == rc and word in lib.sgnn_last_error()


@pytest.mark.parametrize("bad,rc", [
    (dict(lddx=7), -1), (dict(dsv=7), -1), (dict(dsv=1, dsd=69), -1), (dict(grad=None), -1), (dict(stats=None), -1),
    (dict(ws=None), -1), (dict(ws_bytes=16), -2), (dict(B=0), -1), (dict(ldx=7), -1), (dict(dx=None, dw=None), 0),
])
def test_backward_refuses(bad, rc):
    assert backward(_lib(), **bad) == rc


def test_workspace_grows_with_rows_plus_classes():
    lib = _lib()
    need = lib.sgnn_class_xent_workspace_bytes
    assert need(0, 0, 8, 70, 0) == 0 and need(5, 10, 8, 70, 0) == 0
    assert need(0, 10, 1 << 40, 70, 0) == 0 and need(1, 1 << 40, 8, 70, 1) == 0          # the call refuses them
    for dtype in (0, 1):
        for back in (0, 1):
            assert need(dtype, 10, 8, 70, back) > 0
        # far below the logits (4 bytes each, and as much for their gradient)
        assert need(dtype, 65536, 64, 200000, 1) < 65536 * 200000 * 4 / 20


def test_python_layer_needs_gpu_tensors():
    from sgnn_amd import nn
    with pytest.raises(ValueError):
        nn.class_cross_entropy(torch.randn(3, 8), torch.randn(70, 8), torch.zeros(3, dtype=torch.int64))


@pytest.mark.parametrize("B,D,V,pieces", [
    (64, 128, 4096, True), (64, 128, 4095, False), (300, 33, 5001, True), (64, 256, 4096, False), (64, 256, 6000, True),
    (64, 602, 8192, False), (64, 602, 16384, True), (32, 1433, 65536, False), (512, 256, 4096, False),
    (512, 1433, 8192, False), (512, 1433, 16384, True), (4096, 1433, 4096, False), (4096, 602, 4096, True),
])
def test_stacked_heads_in_pieces_where_that_is_faster(B, D, V, pieces):
    from sgnn_amd.stacked import _piecewise_classes
    assert (V >= _piecewise_classes(B, D)) is pieces


def test_rows_that_count_without_a_class_are_asked_for_in_the_type():
    """SGNN_ALL_ROWS goes with fp32 alone; sizes and refusals are those of fp32 otherwise."""
    from sgnn_amd._lib import ALL_ROWS, BF16, F32
    lib = _lib()
    for back in (0, 1):
        assert (lib.sgnn_class_xent_workspace_bytes(F32 | ALL_ROWS, 100, 50, 5000, back)
                == lib.sgnn_class_xent_workspace_bytes(F32, 100, 50, 5000, back) > 0)
    assert forward(lib, dtype=BF16 | ALL_ROWS) == -4 and b"fp32 only" in lib.sgnn_last_error()
    assert forward(lib, dtype=F32 | ALL_ROWS, B=0) == -1 and b"B > 0" in lib.sgnn_last_error()
    assert forward(lib, dtype=2 | ALL_ROWS) == -1 and b"type" in lib.sgnn_last_error()
