"""Limits and refusals of the row operators (nerfslam/rows.py, ns_embedding_* / ns_layer_norm_*) that need no GPU: every check of arguments
comes before the first launch."""
import ctypes as C

import pytest
import torch

from nerfslam import rows
from nerfslam._lib import NerfSlamHipError, lib

P = C.c_void_p(4096)          # an address that no refused call may touch
L = C.c_long


def _refused(rc, word):
    assert rc == -1, rc
    assert word in lib().ns_last_error().decode(), lib().ns_last_error()


def test_a_bias_alone_is_checked_as_a_weight_is():
    x, s = torch.zeros(3, 4), torch.zeros(3)
    for bias, word in ((torch.zeros(3), r"\[4\]"), (torch.zeros(4).half(), "bias is torch.float16"), (torch.zeros(8)[::2], "contiguous")):
        with pytest.raises(NerfSlamHipError, match=word):
            rows.layer_norm_backward(x, x, s, s, None, bias)
    with pytest.raises(NerfSlamHipError, match="one dtype"):
        rows.layer_norm_backward(x.half(), x.half(), s, s, torch.zeros(4), torch.zeros(4).half())
    with pytest.raises(NerfSlamHipError, match="no CPU fallback"):
        rows.layer_norm_backward(x, x, s, s, None, torch.zeros(4))
    f = lib()
    # a bias gradient of many rows needs the workspace, without a weight too; a weight alone has no gradient to go to
    _refused(f.ns_layer_norm_backward(P, L(4), P, L(4), P, P, None, 2, P, None, P, 2, L(3000), 4, P, C.c_size_t(0), None), "workspace")
    _refused(f.ns_layer_norm_backward(P, L(4), P, L(4), P, P, None, 2, P, None, P, 2, L(3000), 4, None, C.c_size_t(1 << 30), None), "workspace")
    _refused(f.ns_layer_norm_backward(P, L(4), P, L(4), P, P, P, 2, P, None, None, 2, L(3), 4, P, C.c_size_t(0), None), "together")
    _refused(f.ns_layer_norm_backward(P, L(4), P, L(4), P, P, None, 2, P, P, None, 2, L(3), 4, P, C.c_size_t(0), None), "together")
    _refused(f.ns_layer_norm_backward(P, L(4), P, L(4), P, P, None, 2, P, None, C.c_void_p(4097), 2, L(3), 4, P, C.c_size_t(0), None), "aligned")


def test_the_largest_gradients_grids():
    """f32 rows of 65536 columns, 2^25 of them (one row expanded along the leading axis): the sums' grid would have 65536 shares x 256 pieces of the
    columns x 256 threads = 2^32 threads, one more than a launch takes.  Refused by its shape; the neighbours are sized as before."""
    f, big, z = lib(), C.c_size_t(1 << 60), C.c_size_t(0)
    size = f.ns_embedding_backward_workspace_bytes
    for n, cols in ((1 << 25, 65536), (1 << 25, 65281), ((1 << 25) - 511, 65536)):
        _refused(f.ns_embedding_backward(P, L(0), 2, P, 0, P, 2, L(n), L(1), cols, C.c_float(1), P, big, None), "2^25 - 512")
        assert size(L(n), L(1), cols, 2) == 0
    for n, cols, dtype in (((1 << 25) - 512, 65536, 2), (1 << 25, 65280, 2), (1 << 25, 65536, 1), (1 << 25, 65536, 3)):
        assert size(L(n), L(1), cols, dtype) > 8 * n
        _refused(f.ns_embedding_backward(P, L(0), dtype, P, 0, P, 2, L(n), L(1), cols, C.c_float(1), P, z, None), "workspace")


def test_every_refusal_is_the_frameworks_error():
    x, ids = torch.zeros(6, 4), torch.zeros(2, 3, dtype=torch.int64).t()
    for call in (lambda: rows.embedding(x, ids), lambda: rows.embedding_backward(torch.zeros(3, 2, 4), ids, 5)):
        with pytest.raises(NerfSlamHipError, match="ids must be contiguous"):
            call()
