"""What the classifier loss and the orthogonalised update refuse, before anything is launched: no GPU needed.  Addresses are
made up and never read."""
import ctypes

import pytest

from tbb_test_amd import capi

P = 1 << 20  # an aligned address
BF, F = capi.MI_BF16, capi.MI_F32
PLENTY = 1 << 60


def refused(name, args, words):
    lib = capi.lib()
    assert getattr(lib, name)(*args) == -1
    text = lib.mi_last_error().decode()
    assert words in text, text


def changed(args, i, value):
    return args[:i] + (value,) + args[i + 1:]


FORWARD = (BF, 4, 100, 64, P, 64, P, 64, None, P, P, P, P, PLENTY, None)
BACKWARD = (BF, 4, 100, 64, P, 64, P, 64, P, 100, None, P, P, None, P, 64, BF, P, 64, None, P, PLENTY, None)
ORTHO = (F, 2, 10, 20, P, 20, 200, P, 20, 200, 5, P, PLENTY, None)
UPDATE = (2, 10, 20, P, P, P, P, P, 200, 400, 2, 0.1, 1.0, 0.0, 0.9, 1, 5, P, PLENTY, None)


@pytest.mark.parametrize("i,value,words", [
    (0, 7, "dtype"), (1, 0, "M, V and K"), (2, -1, "M, V and K"), (3, 0, "M, V and K"), (2, (1 << 21) + 1, "2097152"),
    (4, None, "null"), (5, 63, "ldx"), (6, None, "null"), (7, 63, "ldw"), (9, None, "null"), (10, None, "null"),
    (11, None, "null"), (12, None, "null workspace"), (12, P + 16, "256-byte"), (13, 100, "needed")])
def test_xent_forward(i, value, words):
    refused("mi_xent_forward", changed(FORWARD, i, value), words)


@pytest.mark.parametrize("i,value,words", [
    (0, 2, "dtype"), (1, 0, "M, V and K"), (4, None, "null"), (5, 1, "ldx"), (6, None, "null"), (7, 1, "ldw"), (9, 99, "ldwt"),
    (11, None, "null"), (12, None, "null"), (14, None, "null"), (15, 63, "lddx"), (16, 5, "dw_dtype"), (17, None, "null"),
    (18, 63, "lddw"), (20, None, "null workspace"), (20, P + 128, "256-byte"), (21, 0, "needed")])
def test_xent_backward(i, value, words):
    refused("mi_xent_backward", changed(BACKWARD, i, value), words)


def test_xent_backward_of_an_fp32_model():
    refused("mi_xent_backward", changed(BACKWARD, 0, F), "dw_dtype must be MI_F32 for an fp32 model")
    refused("mi_xent_backward", changed(changed(BACKWARD, 0, F), 16, F), "Wt is for bf16 models")


@pytest.mark.parametrize("i,value,words", [
    (0, 3, "in_dtype"), (1, 0, "batch"), (1, 4097, "batch"), (2, 0, "rows"), (3, 65537, "65536"), (4, None, "null"),
    (5, 19, "ldg"), (6, -1, "strideG"), (7, None, "null"), (8, 19, "ldo"), (9, 199, "strideO"), (10, 0, "steps"),
    (10, 17, "steps"), (11, None, "null workspace"), (11, P + 1, "256-byte"), (12, 1000, "needed")])
def test_orthogonalize(i, value, words):
    refused("mi_orthogonalize", changed(ORTHO, i, value), words)


@pytest.mark.parametrize("i,value,words", [
    (0, 0, "batch"), (1, 0, "rows"), (2, -4, "rows"), (3, None, "null"), (6, None, "null"), (7, None, "null"),
    (8, 199, "layer_stride"), (9, 199, "replica_stride"), (10, 0, "R must"), (16, 0, "steps"), (17, None, "null workspace"),
    (18, 1000, "needed")])
def test_ortho_update(i, value, words):
    refused("mi_ortho_update_raw", changed(UPDATE, i, value), words)


def test_workspace_sizes():
    lib = capi.lib()
    f, b = ctypes.c_size_t(), ctypes.c_size_t()
    for dtype in (BF, F):
        assert lib.mi_xent_workspace(dtype, 300, 5000, 100, ctypes.byref(f), ctypes.byref(b)) == 0
        assert 0 < f.value < 1 << 30 and 0 < b.value < 1 << 31
        assert lib.mi_xent_workspace(dtype, 300, 5000, 100, None, None) == 0
    refused("mi_xent_workspace", (9, 1, 1, 1, None, None), "dtype")
    refused("mi_xent_workspace", (BF, 1, 0, 1, None, None), "M, V and K")
    assert lib.mi_ortho_workspace(3, 100, 200, ctypes.byref(f)) == 0 and f.value >= 3 * 100 * 200 * 10
    refused("mi_ortho_workspace", (1, 1, 1, None), "null result")
    refused("mi_ortho_workspace", (1, 1 << 17, 1, ctypes.byref(f)), "65536")
