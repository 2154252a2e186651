"""Refusals of the row operators (nerfslam/rows.py, ns_embedding_* / ns_layer_norm_*), which need no GPU: every check of arguments comes
before the first launch."""
import ctypes as C

import pytest
import torch

from nerfslam import rows
from nerfslam._lib import NerfSlamHipError, lib

P = C.c_void_p(4096)          # an address that no refused call may touch
L = C.c_long


def _refused(rc, word, status=-1):
    assert rc == status, rc
    assert word in lib().ns_last_error().decode(), lib().ns_last_error()


def test_cpu_tensors_are_refused():
    x, ids = torch.zeros(3, 4), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: rows.embedding(x, ids), lambda: rows.embedding_backward(x, ids, 5), lambda: rows.layer_norm(x),
                 lambda: rows.layer_norm_backward(x, x, torch.zeros(3), torch.zeros(3))):
        with pytest.raises(NerfSlamHipError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("call,word", [
    (lambda x, i: rows.embedding(x.double(), i), "float64"),
    (lambda x, i: rows.embedding(x[0], i), "rows, D"),
    (lambda x, i: rows.embedding(x, i.float()), "int32 or int64"),
    (lambda x, i: rows.embedding(x, i.expand(2, 3).t()), "contiguous"),
    (lambda x, i: rows.embedding(x.t(), i), "contiguous"),
    (lambda x, i: rows.embedding_backward(x, i[:2], 5), "does not match"),
    (lambda x, i: rows.embedding_backward(x, i, -1), "rows"),
    (lambda x, i: rows.embedding_backward(x, i, 5, dtype=torch.float16), "own dtype"),
    (lambda x, i: rows.embedding_backward(x.half(), i, 5, dtype=torch.bfloat16), "own dtype"),
    (lambda x, i: rows.layer_norm(x.int()), "int32"),
    (lambda x, i: rows.layer_norm(x, torch.ones(3)), r"\[4\]"),
    (lambda x, i: rows.layer_norm(x, torch.ones(4).half()), "float16"),
    (lambda x, i: rows.layer_norm(x.half(), torch.ones(4).half(), torch.ones(4)), "one dtype"),
    (lambda x, i: rows.layer_norm(x, torch.ones(8)[::2]), "contiguous"),
    (lambda x, i: rows.layer_norm(torch.zeros(4, 6, 8)[:, :3].transpose(0, 1)), "constant stride"),
    (lambda x, i: rows.layer_norm(torch.tensor(1.0)), "axis"),
    (lambda x, i: rows.layer_norm(torch.empty((1, 2 ** 32 + 4), device="meta")), "65536"),       # (not cut to 4 columns)
    (lambda x, i: rows.embedding(torch.empty((3, 65537), device="meta"), i), "65536"),
    (lambda x, i: rows.layer_norm_backward(x.half(), x, torch.zeros(3), torch.zeros(3)), "does not match"),
    (lambda x, i: rows.layer_norm_backward(x[:2], x, torch.zeros(3), torch.zeros(3)), "does not match"),
    (lambda x, i: rows.layer_norm_backward(x, x, torch.zeros(4), torch.zeros(3)), "mean"),
    (lambda x, i: rows.layer_norm_backward(x, x, torch.zeros(3), torch.zeros(3).half()), "rstd"),
])
def test_arguments_are_checked_before_the_device(call, word):
    with pytest.raises(RuntimeError, match=word):
        call(torch.zeros(3, 4), torch.zeros(3, dtype=torch.int64))


@pytest.mark.parametrize("make,want", [
    (lambda: torch.zeros(6, 8), (6, 8)), (lambda: torch.zeros(6, 8)[:, 2:5], (6, 8)), (lambda: torch.zeros(2, 3, 8)[..., :4], (6, 8)),
    (lambda: torch.zeros(8).expand(6, 8), (6, 0)), (lambda: torch.zeros(8), (1, 8)), (lambda: torch.zeros(6, 8)[::2], (3, 16)),
    (lambda: torch.zeros(4, 1, 5, 8)[:, :, 0], (4, 40)), (lambda: torch.zeros(0, 8), (0, 8)), (lambda: torch.zeros(1, 1, 8), (1, 8)),
    (lambda: torch.zeros(6, 1).expand(6, 1), (6, 1)), (lambda: torch.zeros(2, 6, 1)[0].t().t(), (6, 1)),
])
def test_row_strides(make, want):
    assert rows._rows_of("t", "x", make()) == want


def test_abi_refusals():
    f = lib()
    z = C.c_size_t(0)
    _refused(f.ns_embedding_forward(None, L(4), P, 0, P, 1, L(3), L(5), 4, C.c_float(1), None), "null pointer")
    _refused(f.ns_embedding_forward(P, L(4), None, 0, P, 1, L(3), L(5), 4, C.c_float(1), None), "null pointer")
    _refused(f.ns_embedding_forward(P, L(4), P, 0, P, 7, L(3), L(5), 4, C.c_float(1), None), "dtype")
    _refused(f.ns_embedding_forward(P, L(-1), P, 0, P, 1, L(3), L(5), 4, C.c_float(1), None), "bad shape")
    _refused(f.ns_embedding_forward(P, L(4), P, 0, P, 1, L(-3), L(5), 4, C.c_float(1), None), "bad shape")
    _refused(f.ns_embedding_forward(P, L(4), P, 0, P, 1, L((1 << 25) + 1), L(5), 4, C.c_float(1), None), "2^25")
    _refused(f.ns_embedding_forward(P, L(4), P, 0, P, 1, L(3), L(1 << 31), 4, C.c_float(1), None), "2^31")
    _refused(f.ns_embedding_forward(P, L(4), P, 0, P, 1, L(3), L(5), 0, C.c_float(1), None), "bad shape")
    _refused(f.ns_embedding_forward(P, L(4), P, 0, P, 1, L(3), L(5), 65537, C.c_float(1), None), "65536")
    assert f.ns_embedding_forward(None, L(4), None, 0, None, 1, L(0), L(5), 4, C.c_float(1), None) == 0        # nothing to do

    big = C.c_size_t(1 << 40)
    _refused(f.ns_embedding_backward(P, L(4), 1, P, 0, None, 1, L(3), L(5), 4, C.c_float(1), P, big, None), "null pointer")
    _refused(f.ns_embedding_backward(P, L(4), 1, P, 0, P, 1, L(50000), L(5), 4, C.c_float(1), None, big, None), "null pointer")
    _refused(f.ns_embedding_backward(P, L(4), 1, P, 0, P, 3, L(3), L(5), 4, C.c_float(1), P, big, None), "grad dtype")
    _refused(f.ns_embedding_backward(P, L(4), 2, P, 0, P, 1, L(3), L(5), 4, C.c_float(1), P, big, None), "grad dtype")
    _refused(f.ns_embedding_backward(P, L(4), 1, P, 0, P, 1, L(50000), L(5), 4, C.c_float(1), P, z, None), "workspace")
    _refused(f.ns_embedding_backward(P, L(4), 1, P, 0, P, 1, L(3), L(5), 4, C.c_float(1), C.c_void_p(4100), big, None), "alignment")
    _refused(f.ns_embedding_backward(P, L(4), 1, P, 0, P, 1, L((1 << 25) + 1), L(5), 4, C.c_float(1), P, big, None), "2^25")
    _refused(f.ns_embedding_backward(P, L(4), 1, P, 0, P, 1, L(3), L((1 << 27) + 1), 4, C.c_float(1), P, big, None), "2^27")
    _refused(f.ns_embedding_backward(P, L(4), 1, P, 0, P, 1, L(3), L((1 << 26) + 1), 257, C.c_float(1), P, big, None), "2^27")
    assert f.ns_embedding_backward(None, L(4), 1, None, 0, None, 1, L(3), L(0), 4, C.c_float(1), None, z, None) == 0

    odd = C.c_void_p(4097)
    _refused(f.ns_embedding_forward(odd, L(4), P, 0, P, 1, L(3), L(5), 4, C.c_float(1), None), "aligned")
    _refused(f.ns_embedding_forward(P, L(4), C.c_void_p(4100), 1, P, 1, L(3), L(5), 4, C.c_float(1), None), "aligned")
    _refused(f.ns_embedding_backward(P, L(4), 1, P, 0, C.c_void_p(4098), 2, L(3), L(5), 4, C.c_float(1), P, big, None), "aligned")
    e = C.c_float(1e-5)
    _refused(f.ns_layer_norm_forward(odd, L(4), None, None, 2, P, None, None, 2, L(3), 4, e, None), "aligned")
    _refused(f.ns_layer_norm_backward(P, L(4), P, L(4), P, C.c_void_p(4098), P, 2, P, P, P, 2, L(3), 4, P, big, None), "aligned")
    _refused(f.ns_layer_norm_forward(None, L(4), None, None, 2, P, None, None, 2, L(3), 4, e, None), "null pointer")
    _refused(f.ns_layer_norm_forward(P, L(4), None, None, 2, P, P, None, 2, L(3), 4, e, None), "together")
    _refused(f.ns_layer_norm_forward(P, L(4), P, P, 1, P, P, P, 2, L(3), 4, e, None), "weight dtype")
    _refused(f.ns_layer_norm_forward(P, L(4), P, P, 3, P, P, P, 1, L(3), 4, e, None), "weight dtype")
    _refused(f.ns_layer_norm_forward(P, L(4), P, P, 2, P, P, P, 2, L(3), 16385, e, None), "16384")
    _refused(f.ns_layer_norm_forward(P, L(4), P, P, 2, P, P, P, 2, L(-1), 4, e, None), "bad shape")
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        _refused(f.ns_layer_norm_forward(P, L(4), P, P, 2, P, P, P, 2, L(3), 4, C.c_float(bad), None), "eps")
    assert f.ns_layer_norm_forward(None, L(4), None, None, 2, None, None, None, 2, L(0), 4, e, None) == 0

    _refused(f.ns_layer_norm_backward(P, L(4), P, L(4), P, None, P, 2, P, P, P, 2, L(3), 4, P, big, None), "null pointer")
    _refused(f.ns_layer_norm_backward(P, L(4), P, L(4), P, P, P, 2, P, None, P, 2, L(3), 4, P, big, None), "together")
    _refused(f.ns_layer_norm_backward(P, L(4), P, L(4), P, P, P, 2, P, P, P, 2, L(3000), 4, P, z, None), "workspace")
    _refused(f.ns_layer_norm_backward(P, L(4), P, L(4), P, P, P, 2, P, P, P, 2, L(3), 0, P, big, None), "bad shape")
    _refused(f.ns_layer_norm_backward(P, L(4), P, L(4), P, P, P, 3, P, P, P, 2, L(3), 4, P, big, None), "weight dtype")


def test_workspace_sizes():
    f = lib()
    emb, ln = f.ns_embedding_backward_workspace_bytes, f.ns_layer_norm_backward_workspace_bytes
    assert emb(L(0), L(5), 4, 1) == 0 and ln(L(0), 4, 2) == 0
    assert emb(L(1), L(1000), 64, 2) == 0                    # (short lists need none)
    for n in (8192, 8193, 1 << 20):
        assert emb(L(n), L(1000), 64, 2) >= 8 * n and emb(L(n), L(1000), 64, 3) % 16 == 0
    assert emb(L(1 << 25), L(1 << 19), 65536, 1) > 2 ** 31          # (no 32-bit arithmetic in it)
    assert ln(L(512), 64, 2) == 0 and ln(L(1000), 64, 2) % 512 == 0 and ln(L(1 << 20), 64, 2) > 0
