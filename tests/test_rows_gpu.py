"""Row operators (nerfslam/rows.py) against plain 64-bit forms.

Tolerances: u = 2^-24 is half a step of f32, h(t) = eps(t) / 2 that of an output type.  A sum of m terms in f32 whose longest chain of
additions has k links is off by at most k u sum|terms| (first order); the kernels' row sums have chains of at most 32 terms in a lane,
6 steps across a wave and 16 waves: K = 54, taken as 64.  Every bound below is that arithmetic, written out, times nothing."""
import ctypes as C

import numpy as np
import pytest
import torch

from nerfslam import rows
from nerfslam._lib import NerfSlamHipError, check, graph_capture, lib, ptr, stream_ptr

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
K = 64
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """half a step among the subnormal numbers of a type"""
    return float(torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2)


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device=g.device).to(dtype)


def within(got, want, tol, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    off = (got - want).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(off.max()):.3g}"


# ------------------------------------------------------------------------------------------------ lookup
def make_ids(g, n, v, kind, dtype=torch.int64):
    dev = g.device
    if kind == "one":
        ids = torch.full((n,), v // 2, device=dev)
    elif kind == "skew":          # frequency ~ 1 / rank
        ids = (torch.exp(torch.rand(n, generator=g, device=dev, dtype=torch.float64) * np.log(v + 1.0)).floor().long() - 1).clamp(0, max(v - 1, 0))
    elif kind == "sorted":
        ids = torch.sort(torch.randint(0, v, (n,), generator=g, device=dev))[0]
    else:
        ids = torch.randint(0, max(v, 1), (n,), generator=g, device=dev)
    if kind == "pad":
        r = torch.rand(n, generator=g, device=dev)
        ids = torch.where(r < 0.2, torch.full_like(ids, -1), torch.where(r > 0.9, torch.full_like(ids, v + 3), ids))
    if kind == "none":
        ids = torch.full((n,), -1, device=dev)
    return ids.to(dtype)


def lookup64(table, ids, scale):
    v = table.shape[0]
    live = (ids >= 0) & (ids < v)
    out = torch.zeros((*ids.shape, table.shape[1]), dtype=torch.float64, device=table.device)
    out[live] = table[ids[live].long()].double() * scale
    return out


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n,v,d,kind,idt", [
    (1, 1, 1, "even", torch.int32), (1, 100, 64, "even", torch.int64), (3, 5, 7, "pad", torch.int64), (257, 31, 8, "skew", torch.int32),
    (1000, 50, 33, "pad", torch.int32), (100, 7, 771, "even", torch.int64), (65, 300, 1024, "pad", torch.int64),
    (4099, 1000, 32, "sorted", torch.int32), (5, 2, 65536, "even", torch.int32), (1, 3, 5000, "even", torch.int64), (40, 9, 8200, "pad", torch.int64), (17, 3, 5, "none", torch.int64)])
def test_embedding(dev, n, v, d, kind, idt, dtype):
    g = gen(dev, n + d)
    table, ids = randn(g, v, d, dtype=dtype), make_ids(g, n, v, kind, idt)
    for scale in (1.0, 45.25):
        want = lookup64(table, ids, scale).float().to(dtype)       # one f32 product, one rounding: equal, not close
        assert torch.equal(rows.embedding(table, ids, scale), want)


def test_embedding_shapes_strides_and_empty(dev):
    g = gen(dev, 1)
    wide = randn(g, 40, 96, dtype=F16)
    for table in (wide[:, 3:36], wide[::2], wide[5:6], wide[3, 1:33].expand(9, 32)):
        ids = make_ids(g, 30, table.shape[0], "pad").view(2, 3, 5)
        got = rows.embedding(table, ids)
        assert got.shape == (2, 3, 5, table.shape[1]) and got.is_contiguous()
        assert torch.equal(got, lookup64(table, ids, 1.0).to(F16))
    assert rows.embedding(wide, torch.zeros((0, 4), dtype=torch.int64, device=dev)).shape == (0, 4, 96)
    assert rows.embedding(wide, torch.tensor(7, device=dev)).shape == (96,)
    assert not rows.embedding(wide[:0], torch.zeros(4, dtype=torch.int32, device=dev)).any()
    far = torch.tensor([2 ** 40, -2 ** 40, 2 ** 32 + 3, 3], device=dev)       # no 32-bit cut of a 64-bit id
    assert torch.equal(rows.embedding(wide, far), lookup64(wide, far, 1.0).to(F16))


def test_embedding_scales_nothing_into_padded_places(dev):
    table = torch.tensor([[float("inf"), float("nan"), 1.0]], device=dev)
    got = rows.embedding(table, torch.tensor([0, -1, 1], device=dev), scale=float("inf"))
    assert got[0, 0] == float("inf") and got[0, 1].isnan() and not got[1:].any()


# ------------------------------------------------------------------------------------------------ its gradient
def check_grad(got, dout, ids, v, scale, what):
    """row r has m_r terms: any order of adding them in f32 is off by at most (m_r - 1) u sum|terms|, the product with the scale
    by u, the scale itself (f32) by nothing here, the output by half a step"""
    d = dout.shape[-1]
    ids, dout = ids.reshape(-1).long(), dout.reshape(-1, d)
    live = (ids >= 0) & (ids < v)
    key = ids[live]
    s, a = (torch.zeros((v, d), dtype=torch.float64, device=ids.device) for _ in range(2))
    s.index_add_(0, key, dout[live].double())
    a.index_add_(0, key, dout[live].double().abs())
    m = torch.bincount(key, minlength=v).double()[:, None]
    want = s * scale
    tol = (m * U * a * abs(scale)) + (half(got.dtype) * (1 + m * U) + U) * want.abs() + half(got.dtype) * m * U * a * abs(scale) + tiny(got.dtype)
    tol[m[:, 0] == 0] = 0.0
    within(got, want, tol, what)


SIZES = [(1, 1, 1), (1, 40, 16), (15, 3, 5), (16, 3, 8), (17, 3, 8), (33, 1000, 33), (64, 7, 771), (300, 2, 1030), (1000, 64, 32), (1023, 300, 40), (1024, 70000, 6), (1025, 1, 64), (4095, 257, 130), (4096, 20000, 17),
         (5000, 7, 12), (6001, 900, 771),
         (8192, 300, 8), (8193, 300, 8), (8193, 1023, 4), (9000, 1024, 12), (20000, 70000, 3), (40000, 5, 16), (4097, 5000, 2050),
         (8200, 512, 33), (9300, 512, 64), (30000, 64, 3), (12345, 1, 31), (10240, 513, 32), (9100, 1023, 20), (9200, 1024, 20),
         (32768, 60000, 6), (32769, 60000, 6), (16385, 65535, 8), (16384, 65536, 8), (8195, 4000000, 9),
         (20, 600, 9000), (5, 3, 65536), (9000, 30, 3000), (300, 400000, 3), (1, 300000, 4), (4096, 300000, 9)]


@pytest.mark.parametrize("kind", ["even", "skew", "pad"])
@pytest.mark.parametrize("n,v,d", SIZES)
def test_embedding_backward(dev, n, v, d, kind):
    g = gen(dev, n * 7 + d)
    for dtype, grad, idt in ((F32, F32, torch.int64), (F16, F32, torch.int32), (BF16, BF16, torch.int64), (F16, F16, torch.int32)):
        ids, dout = make_ids(g, n, v, kind, idt), randn(g, n, d, dtype=dtype)
        got = rows.embedding_backward(dout, ids, v, scale=0.5, dtype=grad)
        assert got.dtype == grad and got.shape == (v, d)
        check_grad(got, dout, ids, v, 0.5, (n, v, d, kind, dtype, grad))


@pytest.mark.parametrize("n,v,d,kind", [
    (300000, 1, 8, "one"), (70000, 9, 40, "one"), (262144, 512, 32, "sorted"), (100000, 1 << 21, 2, "even"), (8192, 10, 16, "none"),
    (20000, 10, 16, "none"), (1 << 20, 512, 16, "even"), ((1 << 20) + 5, 512, 8, "skew"), (100000, 300, 60, "one"), (5, 1 << 20, 4, "even"), (270000, 3000, 1, "skew"), (12000, 2000, 515, "sorted")])
def test_embedding_backward_extremes(dev, n, v, d, kind):
    """one row that takes everything (its partial rows are joined by one workgroup), rows in the millions, three radix passes' worth
    of keys, nothing but padded places, lists beyond one tile of the sort"""
    g = gen(dev, v + d)
    ids, dout = make_ids(g, n, v, kind), randn(g, n, d, dtype=F16)
    check_grad(rows.embedding_backward(dout, ids, v), dout, ids, v, 1.0, (n, v, d, kind))


def test_embedding_backward_sorts_stably(dev):
    """integers sum exactly in f32 whatever the order; 2^24-sized ones do not: a fixed order gives the same bits on every call, and an
    exact case gives exact sums for every row of a long skewed list"""
    g = gen(dev, 5)
    for n in (700, 5000, 20000, 100000):
        ids = make_ids(g, n, 3000, "skew")
        whole = torch.randint(-8, 9, (n, 24), generator=g, device=dev).to(F16)
        want = torch.zeros((3000, 24), dtype=torch.float64, device=dev).index_add_(0, ids, whole.double())
        assert torch.equal(rows.embedding_backward(whole, ids, 3000).double(), want)
        dout = randn(g, n, 24) * torch.exp(4 * randn(g, n, 1))
        first = rows.embedding_backward(dout, ids, 3000)
        for _ in range(4):
            assert torch.equal(rows.embedding_backward(dout, ids, 3000), first)


def test_embedding_backward_strides_padding_and_empty(dev):
    g = gen(dev, 6)
    wide = randn(g, 500, 96, dtype=BF16)
    ids = make_ids(g, 500, 40, "pad", torch.int32)
    for dout in (wide[:, 5:38], wide[3, :32].expand(500, 32)):
        check_grad(rows.embedding_backward(dout, ids, 40), dout, ids, 40, 1.0, "strided")
    # what lies in padded places is not used, not even a NaN or an infinity
    dout = wide.clone()
    dout[(ids < 0) | (ids >= 40)] = float("nan")
    got = rows.embedding_backward(dout, ids, 40)
    assert torch.equal(got, rows.embedding_backward(wide, ids, 40)) and got.isfinite().all()
    # an infinity stays in its own row and column
    dout[int(torch.nonzero(ids == 7)[0]), 11] = float("inf")
    got = rows.embedding_backward(dout, ids, 40)
    assert got[7, 11] == float("inf") and int((~got.isfinite()).sum()) == 1
    # many axes, no tokens, no rows
    assert torch.equal(rows.embedding_backward(wide.view(5, 100, 96), ids.view(5, 100), 40), rows.embedding_backward(wide, ids, 40))
    assert not rows.embedding_backward(wide[:0], ids[:0], 40).any()
    assert rows.embedding_backward(wide, ids, 0).shape == (0, 96)


@pytest.mark.parametrize("n,v,d", [(50, 300, 8), (9000, 300, 8), (9000, 3000, 8), (40000, 3000, 8)])
def test_embedding_backward_rows_without_tokens_are_zero_whatever_the_scale(dev, n, v, d):
    ids = torch.arange(n, device=dev) % (v // 2) * 2            # the even rows
    got = rows.embedding_backward(torch.ones((n, d), device=dev), ids, v, scale=float("inf"))
    assert not got[1::2].any() and (got[ids.unique()] == float("inf")).all()


def test_embedding_gradient_is_the_difference_of_the_lookup(dev):
    """<dout, lookup(E + s) - lookup(E)> = <grad, s>: the lookup is linear in the table.  Integers make both sides exact."""
    g = gen(dev, 7)
    ids = make_ids(g, 700, 50, "pad")
    table, step = (torch.randint(-9, 10, (50, 20), generator=g, device=dev).float() for _ in range(2))
    dout = torch.randint(-9, 10, (700, 20), generator=g, device=dev).float()
    diff = (rows.embedding(table + step, ids, 2.0) - rows.embedding(table, ids, 2.0)).double()
    assert float((dout.double() * diff).sum()) == float((rows.embedding_backward(dout, ids, 50, scale=2.0).double() * step.double()).sum())


# ------------------------------------------------------------------------------------------------ layer norm
def norm64(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1)
    c = x - mean[..., None]
    rstd = 1.0 / torch.sqrt((c * c).mean(-1) + eps)
    y = c * rstd[..., None]
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, mean, rstd


def check_norm(got, x, w, b, eps, what):
    """The deviations d = x - m1 carry one rounding (u |d|) whatever m1 is; the correction m2 of the mean is a sum: (K + 2) u mean|d|.
    var is a sum of squares (K + 4 links), so rstd is off by half of that and the roundings of the division and the root (4 u each).
    The output is a product of three factors and a sum (4 u of each part) and rounded to its type."""
    y, mean, rstd = got
    wy, wm, wr = norm64(x, w, b, eps)
    d = (x.double() - wm[..., None]).abs()
    md = d.mean(-1)
    m1_off = (K + 2) * U * x.double().abs().mean(-1)         # (m1 is off by this; it enters |x - m1|)
    md1 = md + m1_off
    r_off = ((K + 4) / 2 + 8) * U + wr * wr * m1_off * m1_off
    within(mean, wm, 2 * U * (wm.abs() + m1_off) + 2 * (K + 2) * U * md1, (what, "mean"))
    within(rstd, wr, wr * r_off, (what, "rstd"))
    ww = 1.0 if w is None else w.double().abs()
    part = (wr * 1.0)[..., None] * ww
    bb = 0.0 if b is None else b.double().abs()
    tol = part * (U * (d + m1_off[..., None]) + (K + 4) * U * md1[..., None]) + part * d * (r_off[..., None] + 4 * U) + 2 * U * (bb + wy.abs())
    within(y, wy, tol * (1 + half(y.dtype)) + half(y.dtype) * wy.abs() + tiny(y.dtype), (what, "y"))


COLS = [1, 2, 3, 8, 31, 64, 65, 128, 200, 256, 512, 771, 1024, 1025, 2048, 2500, 4096, 4104, 8192, 9001, 16384]


@pytest.mark.parametrize("d", COLS)
def test_layer_norm(dev, d):
    for dtype, wdtype, n in ((F32, F32, 5), (F16, F32, 37), (F16, F16, 1), (BF16, BF16, 66), (BF16, F32, 3)):
        g = gen(dev, d + n)
        x = (2.0 * randn(g, n, d) + 0.7 * randn(g, 1, d) - 1.0).to(dtype)
        w, b = (1.0 + 0.2 * randn(g, d)).to(wdtype), (0.3 * randn(g, d)).to(wdtype)
        got = rows.layer_norm(x, w, b, eps=1e-5, stats=True)
        assert got[0].dtype == dtype and got[1].dtype == got[2].dtype == F32 and got[1].shape == (n,)
        check_norm(got, x, w, b, 1e-5, (n, d, dtype, wdtype))
        assert torch.equal(rows.layer_norm(x, w, b, eps=1e-5), got[0])           # the form without statistics: the same bits


@pytest.mark.parametrize("n,d", [(100000, 16), (4097 * 32, 64), (70001, 128), (9000, 1024), (5000, 4096)])
def test_layer_norm_many_rows(dev, n, d):
    g = gen(dev, n)
    x, w, b = randn(g, n, d, dtype=F16), randn(g, d), randn(g, d)
    check_norm(rows.layer_norm(x, w, b, stats=True), x, w, b, 1e-5, (n, d))


def test_layer_norm_without_weights_and_shapes(dev):
    g = gen(dev, 2)
    wide = randn(g, 2, 3, 5, 96, dtype=F16)
    w, b = randn(g, 40, dtype=F16), randn(g, 40, dtype=F16)
    with pytest.raises(NerfSlamHipError, match="constant stride"):       # rows 96 apart, then 1440 = 15 x 96 where 5 x 96 follow each other
        rows.layer_norm(wide[:, 1:2, :, :40])
    for x in (wide[..., 7:47], wide[1:, 1:2, :, :40], wide[0, 0, 0, 1:41], wide[0, 0, 0, :40].expand(6, 40)):
        for ww, bb in ((None, None), (w, None), (None, b), (w, b)):
            y, mean, rstd = got = rows.layer_norm(x, ww, bb, eps=1e-3, stats=True)
            assert y.shape == x.shape and y.is_contiguous() and mean.shape == x.shape[:-1]
            check_norm(got, x, ww, bb, 1e-3, tuple(x.shape))
    assert rows.layer_norm(wide[:0]).shape == (0, 3, 5, 96)


def test_layer_norm_keeps_the_spread_of_rows_far_from_zero(dev):
    """|mean| = 4096 spreads: the deviations come out exact to u |d| because what rounding left of the mean is taken out again"""
    g = gen(dev, 3)
    for d in (64, 1000, 5000):
        x = randn(g, 9, d) + 4096.0
        check_norm(rows.layer_norm(x, eps=1e-6, stats=True), x, None, None, 1e-6, d)


def test_layer_norm_bad_values_stay_in_their_row(dev):
    g = gen(dev, 4)
    keep = [i for i in range(12) if i not in (3, 7)]
    for d in (24, 128, 777, 3000):
        x = randn(g, 12, d, dtype=BF16)
        clean = rows.layer_norm(x)
        x[3, d - 1], x[7, 0] = float("nan"), float("inf")
        y, mean, rstd = rows.layer_norm(x, stats=True)
        assert mean[3].isnan() and mean[7] == float("inf") and rstd[3].isnan() and rstd[7].isnan() and mean[keep].isfinite().all() and rstd[keep].isfinite().all()
        assert torch.equal(y[keep], clean[keep]) and y[3].isnan().all() and y[7].isnan().all()
    const = rows.layer_norm(torch.full((4, 100), 3.0, device=dev), stats=True)       # no spread at all
    assert not const[0].any() and torch.allclose(const[2], torch.full((4,), 1e-5, device=dev).rsqrt(), rtol=1e-6)


def norm_backward64(dout, x, mean, rstd, w):
    dout, x, mean, rstd = dout.double(), x.double(), mean.double()[..., None], rstd.double()[..., None]
    h = (x - mean) * rstd
    g = dout if w is None else dout * w.double()
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    flat = (-1, x.shape[-1])
    return dx, (dout * h).reshape(flat).sum(0), dout.reshape(flat).sum(0), g, h


def check_norm_backward(got, dout, x, mean, rstd, w, what):
    """xh carries 2 u, g u; the two row sums K links; dx is rstd times a difference of three (5 u of each).  dw / db: at least 128
    workgroups share the rows once there are that many, so a lane adds at most n / 128 + 1 of them, a workgroup's 32 lanes of one column
    and the workgroups' partial rows (at most 4096, 16 chains of them) follow: n / 128 + 32 + 256 + 16 links."""
    dx, dw, db = got
    ex, ew, eb, g, h = norm_backward64(dout, x, mean, rstd, w)
    r = rstd.double()[..., None]
    mg, mgh = g.abs().mean(-1, keepdim=True), (g * h).abs().mean(-1, keepdim=True)
    tol = r * (6 * U * g.abs() + (K + 8) * U * mg + h.abs() * (K + 12) * U * mgh) + 2 * U * ex.abs()
    within(dx, ex, tol * (1 + half(dx.dtype)) + half(dx.dtype) * ex.abs() + tiny(dx.dtype), (what, "dx"))
    if w is None:
        assert dw is None and db is None
        return
    flat = (-1, x.shape[-1])
    n = dout.reshape(flat).shape[0]
    links = n / 128 + 1 + 32 + 256 + 16
    for name, have, want, size in (("dw", dw, ew, (dout.double() * h).abs().reshape(flat).sum(0) * (links + 4)),
                                   ("db", db, eb, dout.double().abs().reshape(flat).sum(0) * links)):
        assert have.dtype == w.dtype
        within(have, want, size * U * (1 + half(have.dtype)) + half(have.dtype) * want.abs() + tiny(have.dtype), (what, name))


@pytest.mark.parametrize("d", COLS)
def test_layer_norm_backward(dev, d):
    for dtype, wdtype, n in ((F32, F32, 5), (F16, F32, 37), (F16, F16, 1), (BF16, BF16, 66), (BF16, F32, 3), (F32, None, 70), (F32, F32, 512),
                             (BF16, BF16, 511), (F16, F32, 513), (F16, None, 600), (F32, F32, 700)):
        g = gen(dev, d * 3 + n)
        x = (2.0 * randn(g, n, d) + 0.7 * randn(g, 1, d) - 1.0).to(dtype)
        dout = randn(g, n, d, dtype=dtype)
        w = None if wdtype is None else (1.0 + 0.2 * randn(g, d)).to(wdtype)
        _, mean, rstd = rows.layer_norm(x, w, stats=True)
        check_norm_backward(rows.layer_norm_backward(dout, x, mean, rstd, w), dout, x, mean, rstd, w, (n, d, dtype, wdtype))


@pytest.mark.parametrize("n,d,dtype", [(100000, 16, F16), (70001, 128, F16), (9000, 1024, BF16), (3001, 4096, BF16), (2500, 771, F32), (1300, 16384, F16)])
def test_layer_norm_backward_many_rows(dev, n, d, dtype):
    g = gen(dev, n)
    x, dout, w = randn(g, n, d, dtype=dtype), randn(g, n, d, dtype=dtype), randn(g, d)
    _, mean, rstd = rows.layer_norm(x, w, stats=True)
    got = rows.layer_norm_backward(dout, x, mean, rstd, w)
    check_norm_backward(got, dout, x, mean, rstd, w, (n, d))
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(rows.layer_norm_backward(dout, x, mean, rstd, w), got))


def test_layer_norm_backward_strides_broadcast_and_empty(dev):
    g = gen(dev, 8)
    wide, w = randn(g, 30, 96, dtype=F16), randn(g, 40, dtype=F16)
    for x in (wide[:, 7:47], wide[3, 1:41].expand(30, 40)):
        for dout in (wide[:, 50:90], wide[9, 2:42].expand(30, 40)):
            _, mean, rstd = rows.layer_norm(x, w, stats=True)
            check_norm_backward(rows.layer_norm_backward(dout, x, mean, rstd, w), dout, x, mean, rstd, w, "strided")
    x = wide[:0, :40]
    _, mean, rstd = rows.layer_norm(x, w, stats=True)
    dx, dw, db = rows.layer_norm_backward(x, x, mean, rstd, w)
    assert dx.shape == (0, 40) and not dw.any() and not db.any()


def test_layer_norm_gradients_against_differences(dev):
    """d/ds of L(s) = <c, norm(x + s v)> by the five-point difference of the KERNEL's forward, against <dx, v> of the kernel's backward.
    The difference's own error is measured on the 64-bit formula at the same points; rounding adds (1.5 / step) times the bound of one
    forward pass, sum |c| |y| (K + 20) u, and the gradient's bound.  Weight and bias enter linearly: no truncation there."""
    g = gen(dev, 9)
    x, v, c = randn(g, 6, 80), randn(g, 6, 80), randn(g, 6, 80)
    w, b = 1.0 + 0.2 * randn(g, 80), 0.3 * randn(g, 80)
    step = 2.0 ** -5

    def quotient(f):
        return (8 * (f(step) - f(-step)) - (f(2 * step) - f(-2 * step))) / (12 * step)

    def moved(t, s):
        return (t.double() + s * v.double()[:t.shape[0] if t.dim() > 1 else 1].reshape(t.shape if t.dim() > 1 else -1)).float()

    _, mean, rstd = rows.layer_norm(x, w, b, stats=True)
    dx, dw, db = rows.layer_norm_backward(c, x, mean, rstd, w)
    c64 = c.double()
    ex, ew, eb, _, _ = norm_backward64(c, x, *norm64(x, w, b, 1e-5)[1:], w)
    y = norm64(x, w, b, 1e-5)[0]
    room = 1.5 / step * float((c64 * y).abs().sum()) * (K + 20) * U
    for name, t, have, formula in (("x", x, dx, ex), ("w", w, dw, ew), ("b", b, db, eb)):
        direction = (moved(t, 1.0).double() - t.double())
        args = dict(x=x, w=w, b=b)

        def kernel(s):
            a = dict(args, **{name: (t.double() + s * direction).float()})
            return float((c64 * rows.layer_norm(a["x"], a["w"], a["b"]).double()).sum())

        def plain(s):
            a = dict(args, **{name: (t.double() + s * direction).float()})
            return float((c64 * norm64(a["x"], a["w"], a["b"], 1e-5)[0]).sum())

        want = float((formula * direction).sum())
        trunc = abs(quotient(plain) - want)
        off = float((have.double() - formula).abs().max()) * float(direction.abs().sum())
        assert abs(quotient(kernel) - want) <= trunc + room, name
        assert abs(float((have.double() * direction).sum()) - want) <= off + 1e-12 and off <= room, name


# ------------------------------------------------------------------------------------------------ as they are used
def test_a_run_of_them_together(dev):
    """ids -> rows -> norm and back, against 64-bit autograd of the same chain.  The first output is f32 here, so every stage's bound is a
    few hundred u of its own size and the chain's is their sum: 2^-13 of the largest value leaves a factor of three."""
    g = gen(dev, 10)
    v, d = 60, 96
    table, w, b, c = randn(g, v, d), 1.0 + 0.2 * randn(g, d), 0.3 * randn(g, d), randn(g, 4, 250, d)
    ids = make_ids(g, 1000, v, "pad").view(4, 250)
    e = rows.embedding(table, ids, scale=3.0)
    y, mean, rstd = rows.layer_norm(e, w, b, stats=True)
    de, dw, db = rows.layer_norm_backward(c, e, mean, rstd, w)
    dt = rows.embedding_backward(de, ids, v, scale=3.0)
    t64, w64, b64 = (t.double().cpu().requires_grad_(True) for t in (table, w, b))
    i, live = ids.cpu(), ((ids >= 0) & (ids < v)).cpu()
    e64 = torch.where(live[..., None], t64[torch.where(live, i, 0)] * 3.0, torch.zeros((), dtype=torch.float64))
    y64 = torch.nn.functional.layer_norm(e64, (d,), w64, b64, 1e-5)
    (y64 * c.double().cpu()).sum().backward()
    for name, have, want in (("y", y, y64.detach()), ("table", dt, t64.grad), ("w", dw, w64.grad), ("b", db, b64.grad)):
        within(have.cpu(), want, 2.0 ** -13 * float(want.abs().max()), name)


def _chain(table, ids, w, b, c, v):
    e = rows.embedding(table, ids, scale=2.0)
    y, mean, rstd = rows.layer_norm(e, w, b, stats=True)
    de, dw, db = rows.layer_norm_backward(c, e, mean, rstd, w)
    return y, dw, db, rows.embedding_backward(de, ids, v, scale=2.0)


@pytest.mark.parametrize("n,v", [(300, 40), (5000, 30), (9000, 2000), (9000, 200), (40000, 3000)])
def test_captured_and_replayed(dev, n, v):
    """a whole pass in one HIP graph, replayed on new inputs with eager calls and synchronizations in between; two graphs, each with
    its own workspaces, replayed in turn"""
    g = gen(dev, 11)
    d = 64
    w, b = randn(g, d), randn(g, d)
    sets = [dict(table=randn(g, v, d, dtype=F16), ids=make_ids(g, n, v, "pad"), c=randn(g, n, d, dtype=F16)) for _ in range(3)]
    graphs = []
    for k in range(2):
        live = {a: t.clone() for a, t in sets[k].items()}
        _chain(live["table"], live["ids"], w, b, live["c"], v)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with graph_capture(gr):
            out = _chain(live["table"], live["ids"], w, b, live["c"], v)
        graphs.append((gr, live, out))
    for turn in range(4):
        for k, (gr, live, out) in enumerate(graphs):
            s = sets[(turn + k) % 3]
            for a in live:
                live[a].copy_(s[a])
            gr.replay()
            want = _chain(s["table"], s["ids"], w, b, s["c"], v)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, want)), (turn, k)


def test_two_streams_at_once(dev):
    g = gen(dev, 12)
    v, d, n = 500, 128, 9000
    w, b = randn(g, d), randn(g, d)
    sets = [(randn(g, v, d, dtype=BF16), make_ids(g, n, v, "skew"), w, b, randn(g, n, d, dtype=BF16), v) for _ in range(2)]
    want = [_chain(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(_chain(*sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for run in got[k]:
            assert all(torch.equal(x, y) for x, y in zip(run, want[k]))


def test_nothing_is_written_outside_the_outputs(dev):
    """through the C ABI, with the outputs in the middle of larger buffers at an element's alignment"""
    g = gen(dev, 13)
    f = lib()
    L = C.c_long
    for n, v, d in ((37, 11, 33), (9000, 700, 5), (70, 300, 520), (5000, 70, 33), (20000, 2000, 70), (600, 5, 2000)):
        ids = make_ids(g, n, v, "pad", torch.int32)
        x = randn(g, n * d + 1, dtype=F16)[1:]                                  # 2-byte alignment
        table = randn(g, v * d + 1, dtype=F16)[1:]

        def room(count, dtype):
            buf = torch.full((count + 130,), 7.0, dtype=dtype, device=dev)
            return buf, C.c_void_p(buf.data_ptr() + 65 * buf.element_size()), lambda: buf[65:65 + count], \
                lambda: bool((buf[:65] == 7).all()) and bool((buf[65 + count:] == 7).all())

        _, p, inner, ok = room(n * d, F16)
        check(f.ns_embedding_forward(ptr(table), L(d), ptr(ids), 0, p, 1, L(n), L(v), d, C.c_float(1), stream_ptr()), "fwd")
        assert ok() and torch.equal(inner().view(n, d), rows.embedding(table.view(v, d), ids))
        need = f.ns_embedding_backward_workspace_bytes(L(n), L(v), d, 1)
        ws = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device=dev)
        _, p, inner, ok = room(v * d, F16)
        check(f.ns_embedding_backward(ptr(x), L(d), 1, ptr(ids), 0, p, 1, L(n), L(v), d, C.c_float(1), ptr(ws), C.c_size_t(need), stream_ptr()), "bwd")
        assert ok() and bool((ws[need:] == 0x5a).all())
        assert torch.equal(inner().view(v, d), rows.embedding_backward(x.view(n, d), ids, v, dtype=F16))
        w = randn(g, d)
        _, py, iy, oky = room(n * d, F16)
        _, pm, im, okm = room(n, F32)
        _, pr, ir, okr = room(n, F32)
        check(f.ns_layer_norm_forward(ptr(x), L(d), ptr(w), None, 2, py, pm, pr, 1, L(n), d, C.c_float(1e-5), stream_ptr()), "norm")
        y, mean, rstd = rows.layer_norm(x.view(n, d), w, stats=True)
        assert oky() and okm() and okr() and torch.equal(iy().view(n, d), y) and torch.equal(im(), mean) and torch.equal(ir(), rstd)
        need = f.ns_layer_norm_backward_workspace_bytes(L(n), d, 1)
        ws = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device=dev)
        _, px, ix, okx = room(n * d, F16)
        _, pw, iw, okw = room(d, F32)
        _, pb, ib, okb = room(d, F32)
        check(f.ns_layer_norm_backward(ptr(table[:d]), L(0), ptr(x), L(d), ptr(mean), ptr(rstd), ptr(w), 2, px, pw, pb, 1, L(n), d, ptr(ws),
                                       C.c_size_t(need), stream_ptr()), "norm_bwd")
        dx, dw, db = rows.layer_norm_backward(table[:d].expand(n, d), x.view(n, d), mean, rstd, w)
        assert okx() and okw() and okb() and bool((ws[need:] == 0x5a).all())
        assert torch.equal(ix().view(n, d), dx) and torch.equal(iw(), dw) and torch.equal(ib(), db)


def test_offsets_beyond_32_bits(dev):
    """tables, gradients and activations of more than 2^31 elements: the rows at their ends"""
    v, d = 280000, 8192                                            # 2.29e9 elements, 4.6 GB in f16
    table = torch.zeros((v, d), dtype=F16, device=dev)
    g = gen(dev, 14)
    last = randn(g, 64, d, dtype=F16)
    table[-64:] = last
    ids = torch.arange(v - 64, v, device=dev)
    assert torch.equal(rows.embedding(table, ids), last)
    got = rows.embedding_backward(last, ids, v, dtype=F16)
    assert torch.equal(got[-64:], last) and not got[:4096].any() and not got[v // 2:v // 2 + 4096].any() and not got[-128:-64].any()
    del got
    y, mean, rstd = rows.layer_norm(table, stats=True)
    yl, ml, rl = rows.layer_norm(last, stats=True)
    assert torch.equal(y[-64:], yl) and torch.equal(mean[-64:], ml) and torch.equal(rstd[-64:], rl)
    dx, _, _ = rows.layer_norm_backward(y, table, mean, rstd)
    assert torch.equal(dx[-64:], rows.layer_norm_backward(yl, last, ml, rl)[0])
