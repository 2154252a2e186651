"""Row operators (nerfslam/rows.py) where a bound that grows with the number of terms would let a lost term pass: sums of small whole
numbers, which f32 holds exactly in any order, so that the answer is EQUAL to the 64-bit one or wrong; and random rows by the thousand
against 64 bits for every shape of the norm's row loop.  No term is zero: leaving out any one of them changes every column it is in."""
import ctypes as C

import pytest
import torch

from nerfslam import rows
from nerfslam._lib import check, graph_capture, lib, ptr, stream_ptr
from test_rows_gpu import BF16, F16, F32, U, check_norm, check_norm_backward, gen, half, make_ids, norm64, randn, tiny, within

pytestmark = pytest.mark.gpu


def whole(g, shape, most, dtype):
    """whole numbers of either sign, 1 .. most in size"""
    f = torch.randint(1, most + 1, shape, generator=g, device=g.device).float()
    return (f * (torch.randint(0, 2, shape, generator=g, device=g.device) * 2 - 1)).to(dtype)


def grad64(dout, ids, v):
    """the gradient in 64 bits, and the sum of its terms' sizes.  Rows with many tokens are summed slice by slice of the sorted list: scattered
    additions onto one row take the device minutes."""
    s, a = (torch.zeros((v, dout.shape[-1]), dtype=torch.float64, device=ids.device) for _ in range(2))
    key, order = torch.sort(torch.where((ids >= 0) & (ids < v), ids, torch.full_like(ids, v)).long())
    count = torch.bincount(key, minlength=v + 1)[:v]
    first = torch.cumsum(count, 0) - count
    hot = torch.nonzero(count > 256)[:, 0]
    for r, at, m in zip(hot.tolist(), first[hot].tolist(), count[hot].tolist()):
        d = dout[order[at:at + m]].double()
        s[r], a[r] = d.sum(0), d.abs().sum(0)
    rest = key < v
    rest[rest.clone()] = count[key[rest]] <= 256
    key, d = key[rest], dout[order[rest]].double()
    return s.index_add_(0, key, d), a.index_add_(0, key, d.abs())


def check_whole(dout, ids, v):
    want, size = grad64(dout, ids, v)
    assert float(size.max() if size.numel() else 0.0) < 2.0 ** 24           # every partial sum is exact, whatever the order
    for dtype in {F32, dout.dtype}:
        got = rows.embedding_backward(dout, ids, v, scale=0.5, dtype=dtype)
        assert torch.equal(got, (want * 0.5).float().to(dtype)), (tuple(dout.shape), v, dtype)


def place(dev, counts, n, seed):
    """n ids: counts[r] of row r, the rest padded places, in random order"""
    ids = torch.full((n,), -1, dtype=torch.int64, device=dev)
    at = 0
    for r, m in counts:
        ids[at:at + m] = r
        at += m
    assert at <= n
    return ids[torch.randperm(n, generator=gen(dev, seed), device=dev)]


# one row takes everything, or all but a few tokens: up to 4096 tokens in one launch; up to 1023 narrow rows as tiles' sums added per row;
# else sorted, where the row's run crosses shares of the list: 4 .. 512 of them in these cases, beyond 64 found by search
ONE = [(4096, 50, 771), (4096, 300000, 9), (8192, 10, 130), (8192, 1, 1000), (8192, 5000, 8), (12000, 2000, 1000), (16384, 1, 264), (33000, 1, 1000),
       (70000, 9, 40), (100000, 300, 60), (300000, 1, 8), (1 << 20, 512, 16), (300000, 1024, 8), (100000, 1030, 60), (70000, 1024, 1), (140000, 3, 512)]


@pytest.mark.parametrize("n,v,d", ONE)
def test_one_row_takes_everything(dev, n, v, d):
    g = gen(dev, n + v + d)
    for dtype in (F16, F32):
        dout = whole(g, (n, d), 8, dtype)
        check_whole(dout, torch.full((n,), v // 2, dtype=torch.int32, device=dev), v)
        ids = make_ids(g, n, v, "pad")                                       # a tenth padded or named by chance, the row the others
        check_whole(dout, torch.where(torch.rand(n, generator=g, device=dev) < 0.9, torch.full_like(ids, v - 1), ids), v)


@pytest.mark.parametrize("n,v,d", [(5000, 20, 12), (9000, 40, 300), (12000, 2000, 40), (33000, 1100, 1000), (100000, 1500, 60), (262144, 512, 32), (262144, 1500, 32)])
def test_a_few_rows_take_most(dev, n, v, d):
    """frequency ~ 1 / rank: runs of every length at once, next to each other in the sorted list"""
    g = gen(dev, n + d)
    dout = whole(g, (n, d), 4, F16)
    for kind in ("skew", "sorted", "pad"):
        check_whole(dout, make_ids(g, n, v, kind), v)
    ids = make_ids(g, n, v, "skew")
    check_whole(dout, torch.where(ids < 3, ids, torch.full_like(ids, -1)), v)


@pytest.mark.parametrize("behind", ["row", "padding", "nothing"])
@pytest.mark.parametrize("before", [0, 1, 100, 255, 256])
def test_runs_that_end_at_the_borders_of_shares(dev, before, behind):
    """1000 f16 columns, 33000 tokens: shares of 256 places.  A run that crosses 1, 2, 63 .. 67 shares' ends, ending just before, at and
    behind such an end; the search for the end of a run begins where 64 shares' beginnings have been looked at"""
    n, v, d = 33000, 1, 1000
    dout = whole(gen(dev, before), (n, d), 8, F16)
    lengths = [m * 256 + k for m in (1, 2, 63, 64, 65, 66, 67) for k in (-1, 0, 1)]
    for i, m in enumerate(lengths if behind != "nothing" else [n - before]):
        counts = [(0, before), (1, m)] + ([(2, n - before - m)] if behind == "row" else [])
        check_whole(dout, place(dev, counts, n, i), 3)


@pytest.mark.parametrize("n", [530001, 1100000])
def test_more_than_1024_shares(dev, n):
    """264 and 257 f16 columns: shares of 512 places, 1036 and 2149 of them, so that a workgroup of the join looks at two and at three"""
    d = 264 if n == 530001 else 257
    g = gen(dev, n)
    dout = whole(g, (n, d), 4, F16)
    ids = make_ids(g, n, 3000, "skew", torch.int32)
    check_whole(dout, ids, 3000)
    check_whole(dout, torch.where(torch.rand(n, generator=g, device=dev) < 0.6, torch.full_like(ids, 1), ids), 3000)      # (600 shares of one row)
    check_whole(dout, torch.randint(0, 5, (n,), generator=g, device=dev), 5)


@pytest.mark.parametrize("n,v,d,kind", [
    (300000, 1, 8, "one"), (70000, 9, 40, "one"), (100000, 300, 60, "one"), ((1 << 20) + 5, 512, 8, "skew"), (1 << 20, 512, 16, "even"), (33000, 1, 1000, "one"),
    (300000, 1030, 8, "one"), (140000, 2, 512, "one"), (4096, 3, 771, "one"), (8192, 3, 130, "one")])
def test_embedding_backward_by_the_length_of_its_chains(dev, n, v, d, kind):
    """The longest chain of additions, whatever the number of tokens of a row: at most 128 places in a lane, then 6 steps across a wave and
    16 waves, then the partial rows: 256 sub-groups that each add every 256th (1 lane per row), or 4 that each add every 4th of
    n / 512 (64 lanes) -- below 128 + 6 + 16 + 256 + n / 2048 + 4 links.  A row of 300000 tokens of size 0.8 may then be off by 8; its sums
    are 550 in size, a lost group of 64 tokens 8."""
    g = gen(dev, v + d)
    ids, dout = make_ids(g, n, v, kind), randn(g, n, d)
    want, size = grad64(dout, ids, v)
    links = 410 + n / 2048
    tol = links * U * size * 0.5 + (half(F32) + U) * want.abs() + tiny(F32)
    within(rows.embedding_backward(dout, ids, v, scale=0.5), want * 0.5, tol, (n, v, d, kind))
    if kind == "one":
        assert bool((want.abs()[v // 2] * 0.5 > tol[v // 2]).float().mean() > 0.8)           # (zeros would not pass)


# ------------------------------------------------------------------------------------------------ layer norm
# every shape of the row loop, with more rows than its workgroups take in one turn
@pytest.mark.parametrize("n,d,dtype", [
    (300000, 3, F32), (270000, 32, F32), (140000, 60, F32), (70001, 128, F32), (40000, 250, F32), (40000, 500, F32), (20000, 771, F32), (10000, 1000, F32),
    (6000, 2000, F32), (3000, 4096, F32), (700, 8192, F32), (700, 16384, F32), (600, 9001, F32),
    (270000, 64, BF16), (9000, 2048, BF16), (5000, 4000, F16), (1300, 8192, BF16), (1300, 16384, F16), (1300, 16384, BF16)])
def test_norm_of_many_rows_both_ways(dev, n, d, dtype):
    g = gen(dev, n + d)
    x = (1.5 * randn(g, n, d) + 0.5 * randn(g, 1, d) + 0.3).to(dtype)
    w, b = 1.0 + 0.1 * randn(g, d), 0.1 * randn(g, d)
    check_norm(rows.layer_norm(x, w, b, stats=True), x, w, b, 1e-5, (n, d, dtype))
    _, mean, rstd = norm64(x, None, None, 1e-5)                              # (not the kernel's own)
    mean, rstd, dout = mean.float(), rstd.float(), randn(g, n, d, dtype=dtype)
    check_norm_backward(rows.layer_norm_backward(dout, x, mean, rstd, w), dout, x, mean, rstd, w, (n, d, dtype))


@pytest.mark.parametrize("n,d,dtype,wdtype", [
    (1, 5, F32, F32), (33, 1024, BF16, F32), (512, 771, F32, F32), (511, 16384, F16, F32), (513, 3, F16, F16), (513, 771, F32, F32), (2500, 771, F32, F32),
    (100000, 16, F16, F32), (70001, 128, F16, F32), (230400, 128, F16, F32), (40000, 500, F32, F32), (9000, 1024, BF16, BF16), (3001, 4096, BF16, F32),
    (3000, 4096, F32, F32), (1300, 16384, F16, F16), (700, 16384, F32, F32)])
def test_weight_gradients_lose_no_row(dev, n, d, dtype, wdtype):
    """mean 0 and rstd 1 as given statistics: dweight = sum dout x, dbias = sum dout, of whole numbers"""
    g = gen(dev, n * 3 + d)
    x, dout = whole(g, (n, d), 3, dtype), whole(g, (n, d), 3, dtype)
    mean, rstd = torch.zeros(n, device=dev), torch.ones(n, device=dev)
    assert 9 * n < 2 ** 24
    _, dw, db = rows.layer_norm_backward(dout, x, mean, rstd, whole(g, (d,), 2, wdtype))
    assert torch.equal(dw, (dout.double() * x.double()).sum(0).float().to(wdtype))
    assert torch.equal(db, dout.double().sum(0).float().to(wdtype))


@pytest.mark.parametrize("n,d,dtype,wdtype", [(7, 40, F32, F32), (300, 771, F16, F32), (512, 5000, BF16, BF16), (700, 33, F16, F16), (5000, 128, F32, F32), (600, 2050, BF16, F32), (0, 24, F32, F32)])
def test_gradients_with_and_without_weight_and_bias(dev, n, d, dtype, wdtype):
    """all four forms that the forward pass takes: dx against the formula, dweight and dbias each where it is asked for, and the same bits
    with and without the other"""
    g = gen(dev, n + d)
    x, dout = (1.5 * randn(g, n, d) + 0.3).to(dtype), randn(g, n, d, dtype=dtype)
    w, b = (1.0 + 0.1 * randn(g, d)).to(wdtype), (0.1 * randn(g, d)).to(wdtype)
    _, mean, rstd = rows.layer_norm(x, w, b, stats=True)
    both = rows.layer_norm_backward(dout, x, mean, rstd, w, b)
    check_norm_backward(both, dout, x, mean, rstd, w, (n, d, "both"))
    alone = rows.layer_norm_backward(dout, x, mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip(both, alone))
    dx, dw, db = rows.layer_norm_backward(dout, x, mean, rstd, None, b)
    check_norm_backward((dx, None, None), dout, x, mean, rstd, None, (n, d, "bias"))
    assert dw is None and db.dtype == wdtype and torch.equal(db, both[2])
    plain = rows.layer_norm_backward(dout, x, mean, rstd)
    assert torch.equal(plain[0], dx) and plain[1] is None and plain[2] is None


@pytest.mark.parametrize("weight,bias", [(True, True), (True, False), (False, True), (False, False)])
def test_gradients_of_each_form_against_autograd(dev, weight, bias):
    """torch's own layer norm in 64 bits on the CPU.  f32 in and out: each output is within a few hundred u of the largest of its kind
    (K links of a row sum, n / 128 + 305 of a column), 2^-13 leaves a factor of ten"""
    g = gen(dev, 21)
    x, dout = 1.5 * randn(g, 600, 100) + 0.3, randn(g, 600, 100)
    w, b = (1.0 + 0.1 * randn(g, 100) if weight else None), (0.1 * randn(g, 100) if bias else None)
    y, mean, rstd = rows.layer_norm(x, w, b, stats=True)
    got = (y, *rows.layer_norm_backward(dout, x, mean, rstd, w, b))
    x64, w64, b64 = (None if t is None else t.double().cpu().requires_grad_(True) for t in (x, w, b))
    y64 = torch.nn.functional.layer_norm(x64, (100,), w64, b64, 1e-5)
    (y64 * dout.double().cpu()).sum().backward()
    for name, have, want in zip(("y", "dx", "dw", "db"), got, (y64.detach(), x64.grad, None if w64 is None else w64.grad, None if b64 is None else b64.grad)):
        if want is not None:
            within(have.cpu(), want, 2.0 ** -13 * float(want.abs().max()), name)


def test_a_bias_alone_writes_nothing_else(dev):
    """through the C ABI: dbias in the middle of a larger buffer, no dweight; and a weight without dbias"""
    g, f, L = gen(dev, 22), lib(), C.c_long
    for n, d in ((37, 33), (600, 40), (3000, 1500)):
        x, dout = randn(g, n, d, dtype=F16), randn(g, n, d, dtype=F16)
        w = randn(g, d)
        _, mean, rstd = rows.layer_norm(x, w, stats=True)
        need = f.ns_layer_norm_backward_workspace_bytes(L(n), d, 1)
        for weight in (None, w):
            ws = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device=dev)
            sums, dx = torch.full((d + 130,), 7.0, device=dev), torch.empty_like(x)
            p = C.c_void_p(sums.data_ptr() + 65 * 4)
            check(f.ns_layer_norm_backward(ptr(dout), L(d), ptr(x), L(d), ptr(mean), ptr(rstd), ptr(weight), 2, ptr(dx),
                                           None if weight is None else p, p if weight is None else None, 1, L(n), d, ptr(ws), C.c_size_t(need),
                                           stream_ptr()), "norm_bwd")
            want = rows.layer_norm_backward(dout, x, mean, rstd, weight, w)
            assert torch.equal(dx, want[0]) and torch.equal(sums[65:65 + d], want[2] if weight is None else want[1])
            assert bool((sums[:65] == 7).all()) and bool((sums[65 + d:] == 7).all()) and bool((ws[need:] == 0x5a).all())


@pytest.mark.parametrize("n,d", [(40, 96), (3000, 96)])
def test_a_bias_alone_captured_and_replayed(dev, n, d):
    """in one launch and with partial rows: replayed on new inputs, eager calls and synchronizations between the replays"""
    g = gen(dev, n)
    b = 0.1 * randn(g, d)
    sets = [(randn(g, n, d, dtype=BF16), randn(g, n, d, dtype=BF16)) for _ in range(3)]

    def both(x, dout):
        y, mean, rstd = rows.layer_norm(x, None, b, stats=True)
        dx, _, db = rows.layer_norm_backward(dout, x, mean, rstd, None, b)
        return y, dx, db

    live = [t.clone() for t in sets[0]]
    both(*live)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with graph_capture(graph):
        out = both(*live)
    for turn in range(4):
        for t, new in zip(live, sets[turn % 3]):
            t.copy_(new)
        graph.replay()
        want = both(*sets[turn % 3])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want)), turn
