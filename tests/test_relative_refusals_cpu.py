"""The backward entry of the relative bias names the argument that is wrong, without a GPU."""
import ctypes

import pytest

import fast_ops_b200._lib as L


def backward(workspace=16, starts=(0, 1, 2, 5), table_dtype=L.FO_F32, dtype=L.FO_BF16):
    lib = L.load()
    s = (ctypes.c_int64 * 3)(8 * 64 * 2, 8 * 64, 64)
    array = None if starts is None else (ctypes.c_int * len(starts))(*starts)
    rc = lib.fo_rel_attn_bwd(*([16] * 13), 1, 2, 8, 8, 64, *([s] * 8), dtype, 0, -1.0, table_dtype, array, 4, 1, 0, workspace,
                             None, None, L.FO_F32, 0.0, 0, 0, 0, None)
    return rc, lib.fo_last_error()


@pytest.mark.parametrize("change,message", [
    (dict(workspace=None), b"null workspace"), (dict(workspace=18), b"workspace must be 16-byte aligned"),
    (dict(workspace=17), b"workspace must be 16-byte aligned"), (dict(workspace=24), b"workspace must be 16-byte aligned"),
    (dict(starts=None), b"null bucket starts"), (dict(table_dtype=L.FO_F16), b"table must be fp32"),
    (dict(dtype=L.FO_F32), b"fp16 or bf16"), (dict(), b"softmax_scale")])
def test_the_message_names_the_argument(change, message):
    rc, error = backward(**change)
    assert rc == -1 and message in error, error


def test_workspace_size_without_starts():
    lib = L.load()
    assert lib.fo_rel_attn_workspace(1, 8, 8, None, 4, 1, 0, 0) == -1 and b"null bucket starts" in lib.fo_last_error()
